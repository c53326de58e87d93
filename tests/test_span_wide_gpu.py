"""The span attention's kernel for many query rows: sizes that are cut for it (tests/test_span_plan.py asserts that they
are), against the closed form in 64 bits.

Tolerance, per output: that of tests/test_span_gpu.py, and what two float16 terms leave of a value. Of a q it is at most
2^-23 of itself, so 2^-23 of a score's terms, and further terms are taken where the rest could pass 2^-24 of a score times
log2 e. Of p * v_scale it is at most 2^-23 of itself, so 2^-23 of sum p |V|, and 2^-26 of the largest one that the row has
in the tile of 32 keys, among those whose V rows are not zeros (a zero row adds exactly nothing).
"""
import numpy as np
import pytest

from openneedle_amd.device import DeviceArray, Graph, Stream, synchronize
from tests.test_evict_gpu import read_rows
from tests.test_span_gpu import EPS, Rows, check, ring_slot, run_shared, run_window, seen, upload

pytestmark = pytest.mark.gpu

# (sequences, kv heads, query heads per kv head, tokens, sinks, window): windows shorter and longer than the piece, one and
# two blocks of rows, groups that do not divide a block's rows, one piece of the keys and many
EDGES = [(16, 8, 4, 40, 3, 40), (40, 8, 3, 43, 4, 90), (20, 8, 16, 9, 0, 150), (40, 8, 3, 50, 70, 1), (16, 8, 2, 130, 0, 64),
         (64, 8, 1, 17, 3, 40), (24, 8, 5, 64, 3, 70), (64, 8, 4, 5, 4, 60)]
LONG = (1, 2, 2, 40, 0, 4000)     # pieces of one or two tiles
PIECE = (32, 8, 2, 40, 0, 301)    # one piece of twelve
# (sequences, kv heads, query heads per kv head, prefix)
PREFIXES = [(40, 1, 4, 700), (17, 2, 3, 700), (9, 2, 4, 30011)]
GRAPH_WINDOW, GRAPH_PREFIX, GRAPH_OUTGROWN = LONG, (40, 2, 2, 700), (1, 2, 8, 300, 0, 3740)


def attend(q, k, v, vs, tiles=None):
    """(output, tolerance) of one query row over rows k, v in 64 bits; vs: the V rows' scales, tiles: the keys' tiles
    (none: as if all were in one, which the bound of the largest weight covers)."""
    hd = q.shape[-1]
    if len(k) == 0:
        return np.zeros(hd), np.zeros(hd)
    q = q.astype(np.float64)
    x = k @ q / np.sqrt(hd)
    p = np.exp(x - x.max())
    p /= p.sum()
    size = (np.abs(k) @ np.abs(q)).max() / np.sqrt(hd)
    score = (np.sqrt(3 * hd) + 16 + 2) * EPS * size + EPS
    tol = (2 * score + (np.sqrt(3 * len(k)) + 8 + 2) * EPS) * (p @ np.abs(v)) + 1e-37
    weight = np.where(v.any(-1), p * np.abs(vs), 0)
    codes = np.abs(v) / np.where(vs == 0, 1, np.abs(vs))[:, None]
    tiles = np.zeros(len(k), int) if tiles is None else tiles
    for t in np.unique(tiles):
        mine = tiles == t
        tol = tol + 2.0 ** -26 * weight[mine].max() * codes[mine].sum(0)
    return p @ v, tol


def check_ring(r, q, positions, sinks, window, got, seqs, kv_heads, tokens, tiled=False):
    """tiled: slot = position, the first row's first key at the start of a tile of 32."""
    cap = r.k.shape[1]
    group = q.shape[2] // r.k.shape[2]
    for s in seqs:
        for i in tokens:
            at = np.array(seen(positions[s] + i, sinks, window), np.int64)
            slots = np.where(at < sinks, at, sinks + (at - sinks) % (cap - sinks))
            for h in kv_heads:
                k, v = r.at(s, slots, h)
                for g in range(h * group, h * group + group):
                    want, tol = attend(q[s, i, g], k, v, r.vs[s, slots, h].astype(np.float64), slots // 32 if tiled else None)
                    check(got[s, i, g], want, tol, f"sequence {s} token {i} head {g}")


def rows_of(rng, shape, hd, extra=0, **kw):
    seqs, kvh, group, count, sinks, window = shape
    return Rows(rng, seqs, sinks + window + count - 1 + extra, kvh, hd, **kw)


def queries(rng, shape, hd):
    seqs, kvh, group, count = shape[:4]
    return rng.normal(size=(seqs, count, kvh * group, hd)).astype(np.float32)


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("shape", EDGES)
def test_ring_edges(hd, shape):
    """New rows stored first; left padding, before the window is full, wraps inside the piece, far positions."""
    seqs, kvh, group, count, sinks, window = shape
    rng = np.random.default_rng(hd + sum(shape))
    r, q = rows_of(rng, shape, hd, extra=window % 3), queries(rng, shape, hd)
    kinds = [0, -count, 1 - count, -2, 1, sinks + 1, window, window + sinks, 5 * window + 7, 12345, 2 ** 31 - 1 - count]
    positions = [kinds[s % len(kinds)] for s in range(seqs)]
    new = tuple(rng.normal(size=(seqs, count, kvh, hd)).astype(np.float32) for _ in "kv")
    got = run_window(r, q, positions, sinks, window, new)
    for s, first in enumerate(positions):
        for i in range(count):
            if first + i >= 0:
                r.put(s, ring_slot(first + i, sinks, r.k.shape[1]), new[0][s, i], new[1][s, i])
    r.same()
    tokens = sorted({0, 1, 2, count // 2, count - 2, count - 1})
    check_ring(r, q, positions, sinks, window, got, range(len(kinds)), (0, kvh - 1), tokens)


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_pieces_and_rows_stored_before(hd):
    """Many pieces of the keys; without new rows the tokens' own are taken from the cache; the second of two layers."""
    rng = np.random.default_rng(hd)
    r, q = rows_of(rng, LONG, hd, extra=7, layers=2, layer=1), queries(rng, LONG, hd)
    for first in (50, 3999, 123456):
        check_ring(r, q, [first], 0, 4000, run_window(r, q, [first], 0, 4000), [0], [0, 1], [0, 17, 39])


def piece(rng, hd, change, q=None, tokens=range(40), kv_heads=(0, 1)):
    """PIECE with rows as `change` leaves them, every sequence alike: token i attends positions i .. i + 300."""
    seqs, kvh = PIECE[:2]
    r = rows_of(rng, PIECE, hd)
    change(r)
    r.push()
    q = queries(rng, PIECE, hd) if q is None else q
    got = run_window(r, q, [300] * seqs, 0, 301)
    check_ring(r, q, [300] * seqs, 0, 301, got, (0, seqs - 1), kv_heads, tokens, tiled=True)
    return got


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("ratio", [1e4, 1e6, 1e8, 1e12, 1e30])
def test_uneven_queries(hd, ratio):
    """Entries of q far above the rest over zero K codes, in some rows only: the other entries' products decide."""
    rng = np.random.default_rng(hd + int(np.log10(ratio)))
    q = queries(rng, PIECE, hd)
    q[:, 3::7, :, 5] = ratio
    q[:, 5] *= 1e-30
    q[:, 6] = 0

    def change(r):
        r.k[:, :, :, 5] = 0
    piece(rng, hd, change, q, tokens=(0, 3, 5, 6, 7, 10, 39))


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("apart", [-110, -60, 20, 60, 90, 110])
@pytest.mark.parametrize("margin", [0, 30000])
def test_extreme_queries_and_k_scales(hd, apart, margin):
    """Queries 2^apart times smaller, K scales as much larger; a slot with scores of 30000."""
    rng = np.random.default_rng(hd + apart + 200)
    q = queries(rng, PIECE, hd)

    def change(r):
        if margin:
            dominant(q, r, 77, margin)
        r.ks *= np.float32(2.0 ** apart)
        q[:] *= np.float32(2.0 ** -apart)
    piece(rng, hd, change, q, tokens=(0, 1, 39))


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("margin", [3, 10, 30, 60, 120])
def test_dominant_slots(hd, margin):
    """Some slots whose scores are `margin` above the rest, with zero V codes in half of the dimensions: there the other
    slots' sums show."""
    rng = np.random.default_rng(hd + margin)
    sign = rng.choice([-1, 1], hd)
    q = (np.abs(queries(rng, PIECE, hd)) * sign).astype(np.float32)

    def change(r):
        for j in (0, 77, 200):
            r.k[:, j] = 127 * sign
            r.ks[:, j] = margin * np.sqrt(hd) / (127 * np.abs(q).sum(-1).mean())
            r.v[:, j, :, ::2] = 0
    piece(rng, hd, change, q, tokens=(0, 1, 39))


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("scales", ["tiny", "huge", "mixed", "zero", "signed"])
def test_v_scales(hd, scales):
    def change(r):
        if scales == "tiny":
            r.vs *= np.float32(2.0 ** -108)
        elif scales == "huge":
            r.vs *= np.float32(2.0 ** 118)
        elif scales == "mixed":
            r.vs[:, :160] *= np.float32(2.0 ** -100)
            r.vs[:, 100] = 2.0 ** 90
            r.vs[:, 200:] *= np.float32(2.0 ** -30)
        elif scales == "zero":
            r.vs[:, :200] = 0
        else:
            r.vs[:, ::3] *= -1
            r.ks[:, ::2] *= -1
    piece(np.random.default_rng(50 + hd), hd, change, tokens=(0, 1, 20, 39))


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_non_finite_input(hd):
    """As for few rows: a head with an infinity or NaN in its query yields zeros and leaves the others alone; an infinite
    V scale gives infinities of the codes' signs (NaN for a zero code) to the rows that attend it, of its kv head."""
    rng = np.random.default_rng(8 + hd)
    seqs, kvh, group, count, sinks, window = PIECE
    r, q = rows_of(rng, PIECE, hd), queries(rng, PIECE, hd)
    q[0, 0, 0, 3] = np.nan
    q[0, 1, 1, 9] = np.inf
    q[0, 39, 2, hd - 1] = -np.inf
    first = [300] * seqs
    got = run_window(r, q, first, 0, 301)
    for i, h in ((0, 0), (1, 1), (39, 2)):
        assert not got[0, i, h].any()
        q[0, i, h] = 0  # and what any finite query gives, for the check below
    again = run_window(r, q, first, 0, 301)
    for i, h in ((0, 0), (1, 1), (39, 2)):
        got[0, i, h] = again[0, i, h]
    np.testing.assert_array_equal(got, again)
    check_ring(r, q, first, 0, 301, got, [0, 1], [0, 1], [0, 1, 2, 39])
    r.vs[0, 20, 1] = np.inf  # attended by tokens 0 to 20 only
    r.v[0, 20, 1, 3] = 0
    r.push()
    got = run_window(r, q, first, 0, 301)
    codes = r.v[0, 20, 1]
    want = np.where(codes == 0, np.nan, np.where(codes > 0, np.inf, -np.inf))
    for i in (0, 20):
        for h in (2, 3):
            np.testing.assert_array_equal(got[0, i, h], want)
    check_ring(r, q, first, 0, 301, got, [0], [1], [21, 39])
    check_ring(r, q, first, 0, 301, got, [0, 1], [0], [0, 20, 39])


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("value", [np.nan, np.inf, 3e38, 1e-38])
def test_what_is_not_attended_does_not_matter(hd, value):
    """Slots outside the window hold scales that are infinite, NaN or at the ends of the range."""
    rng = np.random.default_rng(6)
    seqs, kvh, group, count, sinks, window = shape = EDGES[0]
    r, q = rows_of(rng, shape, hd, extra=90), queries(rng, shape, hd)
    cap = r.k.shape[1]
    positions = [(0, 20, 300, 501)[s % 4] for s in range(seqs)]
    for s, first in enumerate(positions):
        live = {ring_slot(j, sinks, cap) for i in range(count) for j in seen(first + i, sinks, window)}
        dead = [j for j in range(cap) if j not in live]
        assert dead
        r.ks[s, dead] = value
        r.vs[s, dead] = value
    r.push()
    got = run_window(r, q, positions, sinks, window)
    check_ring(r, q, positions, sinks, window, got, range(4), (0, 7), (0, 1, 20, 38, 39))


def test_unaligned_buffers():
    """q and the output start at any float."""
    rng = np.random.default_rng(33)
    seqs, kvh, group, count, sinks, window = shape = EDGES[1]
    r, q = rows_of(rng, shape, 64), queries(rng, shape, 64)
    d_n, big = upload([299] * seqs, np.int32), [DeviceArray(q.nbytes + 16) for _ in range(2)]
    for off in (4, 8, 12):
        d_q, d_o = (b.view(off, q.nbytes) for b in big)
        d_q.upload(q)
        r.kv.attention_window(0, d_q, d_o, kvh * group, count, d_n, sinks, window)
        synchronize()
        check_ring(r, q, [299] * seqs, sinks, window, d_o.to_host(np.float32, q.shape), [0], [0, kvh - 1], (0, 17, count - 1))


def test_same_results_every_time():
    rng = np.random.default_rng(30)
    for shape, first in ((PIECE, 300), (LONG, 5000)):
        r, q = rows_of(rng, shape, 128), queries(rng, shape, 128)
        one = run_window(r, q, [first] * shape[0], 0, shape[5])
        for _ in range(3):
            np.testing.assert_array_equal(run_window(r, q, [first] * shape[0], 0, shape[5]), one)


# ---- a shared prefix --------------------------------------------------------------------------------------------------
def shared(rng, shape, hd, change=None, q=None, seqs=(0, 1, -1), tiled=True):
    n, kvh, group, length = shape
    prefix, r = Rows(rng, 1, length + 3, kvh, hd), Rows(rng, n, 70, kvh, hd)
    if change:
        change(prefix, r)
        prefix.push()
        r.push()
    q = rng.normal(size=(n, kvh * group, hd)).astype(np.float32) if q is None else q
    lengths = rng.integers(1, 70, n)
    lengths[1] = 0
    got = run_shared(r, prefix, length, q, 70, lengths)
    for h in range(kvh):
        pk, pv = prefix.at(0, range(length), h)
        for s in seqs:
            k, v = r.at(s, range(lengths[s]), h)
            both = np.concatenate([pk, k]), np.concatenate([pv, v])
            vs = np.concatenate([prefix.vs[0, :length, h], r.vs[s, :lengths[s], h]]).astype(np.float64)
            # (the sequences' own slots have exact weights: any tiles cover them)
            tiles = np.concatenate([np.arange(length) // 32, 10 ** 6 + np.arange(lengths[s])])
            for g in range(h * group, h * group + group):
                want, tol = attend(q[s, g], *both, vs, tiles if tiled else None)
                check(got[s, g], want, tol, f"sequence {s} head {g}")


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("shape", PREFIXES)
def test_prefix(hd, shape):
    shared(np.random.default_rng(hd + shape[0]), shape, hd)


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("scales", ["tiny", "huge", "mixed", "zero", "signed", "infinite"])
def test_prefix_v_scales(hd, scales):
    def change(p, r):
        if scales == "tiny":
            p.vs *= np.float32(2.0 ** -108)
            r.vs *= np.float32(2.0 ** -108)
        elif scales == "huge":
            p.vs *= np.float32(2.0 ** 118)
        elif scales == "mixed":
            p.vs[:, :16000] *= np.float32(2.0 ** -100)
            p.vs[:, 10000] = 2.0 ** 90
            r.vs *= np.float32(2.0 ** -30)
        elif scales == "zero":
            p.vs[:, :20000] = 0
        elif scales == "signed":
            p.vs[:, ::3] *= -1
            p.ks[:, ::2] *= -1
        else:  # behind the prefix
            p.vs[:, -3:] = np.inf
            p.ks[:, -2:] = np.nan
    shared(np.random.default_rng(60 + hd), PREFIXES[2], hd, change)


def test_prefix_non_finite_query():
    rng = np.random.default_rng(70)
    n, kvh, group, length = PREFIXES[0]
    prefix, r = Rows(rng, 1, length, kvh, 64), Rows(rng, n, 8, kvh, 64)
    q = rng.normal(size=(n, kvh * group, 64)).astype(np.float32)
    clean = run_shared(r, prefix, length, q, 8, None)
    q[3, 1, 7] = np.nan
    q[39, 3, 0] = -np.inf
    got = run_shared(r, prefix, length, q, 8, None)
    assert not got[3, 1].any() and not got[39, 3].any()
    clean[3, 1] = clean[39, 3] = 0
    np.testing.assert_array_equal(got, clean)


# ---- V scales of a tile far apart ---------------------------------------------------------------------------------------
def dominant(q, rows, at, margin):
    """Slot `at` of every sequence with scores about `margin` above the rest; q gets one sign a dimension."""
    hd = q.shape[-1]
    sign = np.where(np.arange(hd) % 3 == 0, -1, 1)
    q[:] = np.abs(q) * sign
    rows.k[:, at] = 127 * sign
    rows.ks[:, at] = margin * np.sqrt(hd) / (127 * np.abs(q).sum(-1).mean())


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("apart", [8, 12, 16, 20, 24, 30, 36, 60])
def test_the_largest_score_at_a_small_v_scale(hd, apart):
    rng = np.random.default_rng(apart)
    q = queries(rng, PIECE, hd)

    def change(r):
        dominant(q, r, 77, 30)
        r.vs[:, 77] *= np.float32(2.0 ** -apart)
    piece(rng, hd, change, q, tokens=(0, 1, 39))


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("apart", [8, 15, 20, 25, 30, 40, 60, 100, 120])
def test_v_scales_of_keys_that_a_row_does_not_attend(hd, apart):
    """Position 310 is attended by the tokens from 10 on, position 5 by those up to 5; their tiles by all. Both V scales are
    2^apart times the rest's."""
    def change(r):
        r.vs[:, 310] = r.vs[:, 5] = np.float32(0.015 * 2.0 ** apart)
    piece(np.random.default_rng(apart), hd, change, tokens=(0, 5, 6, 9, 10, 39))


@pytest.mark.parametrize("hd", [32, 128])
def test_v_scales_that_change_from_tile_to_tile(hd):
    """The outputs meet weights far larger and far smaller than themselves, in every order."""
    rng = np.random.default_rng(hd)

    def change(r):
        for t, e in enumerate((0, 60, -60, 30, -100, 90, -20, 110, -110, 10, -50)):
            r.vs[:, 32 * t:32 * t + 32] *= np.float32(2.0 ** e)
            r.v[:, 32 * t:32 * t + 32, :, t:t + 1] = 0  # where the tile's own codes are zeros the others show
    piece(rng, hd, change, tokens=(0, 39))


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("at", [0, 40, 170, 299])
@pytest.mark.parametrize("margin", [12, 40, 60])
def test_scores_far_apart_and_v_scales_that_change(hd, at, margin):
    """A slot with scores far ahead, in an early or late tile, whose V row has zeros in half of the dimensions, beside tiles
    of V scales far above and below: tiles far below the row's maximum with scales beyond what it follows."""
    rng = np.random.default_rng(hd + at + margin)
    q = queries(rng, PIECE, hd)

    def change(r):
        dominant(q, r, at, margin)
        r.v[:, at, :, ::2] = 0
        for t, e in enumerate((0, 55, -20, 3, 70, -3, 8, -8, 60, 0, 20)):
            r.vs[:, 32 * t:32 * t + 32] *= np.float32(2.0 ** e)
    piece(rng, hd, change, q, tokens=(0, 1, 39))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("apart", [12, 24, 36])
def test_prefix_the_largest_score_at_a_small_v_scale(hd, apart):
    rng = np.random.default_rng(apart + 1)
    n, kvh, group, length = PREFIXES[2]
    q = rng.normal(size=(n, kvh * group, hd)).astype(np.float32)

    def change(p, r):
        dominant(q, p, 7777, 30)
        p.vs[:, 7777] *= np.float32(2.0 ** -apart)
        r.vs *= np.float32(2.0 ** -apart)
    shared(rng, PREFIXES[2], hd, change, q)


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("apart", [0, 8, 16, 20, 24, 30, 36, 60])
@pytest.mark.parametrize("margin", [0, 30])
def test_v_rows_of_zeros(hd, apart, margin):
    """A V row of zeros as the cache stores it (scale 1), the others' scales 2^apart below; its score is like the others'
    or far ahead of them. Two such rows in a tile, and a row of which only one value is not zero."""
    rng = np.random.default_rng(apart + margin)
    q = queries(rng, PIECE, hd)

    def change(r):
        r.vs *= np.float32(2.0 ** -apart)
        for at in (77, 79, 160, 319):
            if margin and at != 160:
                dominant(q, r, at, margin)
            r.v[:, at] = 0
            r.vs[:, at] = 1
        r.v[:, 78] = 0
        r.v[:, 78, :, hd - 1] = 3
        r.vs[0, 200, 1] = np.nan if apart == 36 else r.vs[0, 200, 1]
        r.v[0, 200, 1] = 0 if apart == 36 else r.v[0, 200, 1]
    got = piece(rng, hd, change, q, tokens=(0, 1, 39), kv_heads=(0,) if apart == 36 else (0, 1))
    if apart == 36:  # zeros with a scale that is no number
        assert np.isnan(got[0, :, 2:4]).all()


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_prefix_v_rows_of_zeros(hd):
    rng = np.random.default_rng(hd)
    n, kvh, group, length = PREFIXES[2]
    q = rng.normal(size=(n, kvh * group, hd)).astype(np.float32)

    def change(p, r):
        dominant(q, p, 7777, 60)
        p.v[:, [7777, 64, 0, 30010]] = 0
        p.vs *= np.float32(2.0 ** -20)
        r.vs *= np.float32(2.0 ** -20)
        p.vs[:, [7777, 64, 0, 30010]] = 1
    shared(rng, PREFIXES[2], hd, change, q)


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_v_scales_of_one(hd):
    """Rows of the scale that rows of zeros have, zeros in all but their last codes."""
    rng = np.random.default_rng(hd)

    def change(r):
        r.vs[:] = 1
        r.v[:, ::5, :, :hd - 1] = 0
        r.v[:, ::5, :, hd - 1] = 1
        r.v[:, ::15] = 0
    piece(rng, hd, change, tokens=(0, 39))


# ---- captured -----------------------------------------------------------------------------------------------------------
def test_graph_replays_match_eager():
    """A window step and a shared-prefix step of the many-row kernel, a recorded step and a cut in place whose list is the
    handle's scratch, captured into one graph and replayed with other inputs. Between the replays eager calls of larger
    sizes on the same handles outgrow the scratch of each."""
    hd, cap, keep = 64, 300, 100
    _, kvh, group, count, sinks, window = GRAPH_WINDOW
    n, _, _, prefix = GRAPH_PREFIX
    heads = kvh * group

    def state():
        rng = np.random.default_rng(1)
        d = dict(ring=rows_of(rng, GRAPH_WINDOW, hd), own=Rows(rng, n, cap, kvh, hd), prefix=Rows(rng, 1, prefix, kvh, hd))
        for name, size in dict(q=count * heads, nk=count * kvh, nv=count * kvh, o=count * heads, q1=n * heads, k1=n * kvh,
                               v1=n * kvh, o1=n * heads, o2=n * heads).items():
            d[name] = DeviceArray(size * hd * 4)
        d["pos"], d["n"], d["w"] = DeviceArray(4), DeviceArray(n * 4), DeviceArray(n * kvh * cap * 4)
        d["big_q"], d["big_o"] = (DeviceArray(GRAPH_OUTGROWN[3] * 8 * heads * hd * 4) for _ in "qo")
        d["big_w"] = DeviceArray(n * kvh * cap * 4)
        return d

    def feed(d, seed):
        rng = np.random.default_rng(seed)
        for name in ("q", "nk", "nv", "q1", "k1", "v1"):
            d[name].upload(rng.normal(size=d[name].nbytes // 4).astype(np.float32))
        d["pos"].upload(rng.integers(0, 9000, 1).astype(np.int32))
        d["n"].upload(rng.integers(50, cap, n).astype(np.int32))
        d["w"].upload(rng.random(n * kvh * cap).astype(np.float32))

    def step(d, stream):
        d["ring"].kv.attention_window(0, d["q"], d["o"], heads, count, d["pos"], sinks, window, stream=stream,
                                      new=(d["nk"], d["nv"]))
        d["own"].kv.attention_shared(0, d["prefix"].kv, prefix, d["q1"], d["o1"], heads, cap, d["n"], stream=stream,
                                     new=(d["k1"], d["v1"]))
        d["own"].kv.attention_weights(0, d["q1"], d["o2"], d["w"], heads, cap, d["n"], stream=stream)
        d["own"].kv.evict(0, d["w"], d["n"], keep, 4, 32, d["w"], d["n"], stream=stream)

    def outgrow(d, stream, i):
        """More query rows and heads, so more records and scores; a larger keep."""
        more = heads * (2, 4, 8, 8)[i]
        d["big_q"].fill(0)
        d["big_w"].fill(0)
        _, _, many, tokens, _, span = GRAPH_OUTGROWN
        d["ring"].kv.attention_window(0, d["big_q"], d["big_o"], kvh * many, tokens, d["pos"], 0, span, stream=stream)
        d["own"].kv.attention_shared(0, d["prefix"].kv, prefix, d["big_q"], d["big_o"], more, cap, stream=stream)
        d["own"].kv.attention_weights(0, d["big_q"], d["big_o"], d["big_w"], more, cap, stream=stream)
        d["own"].kv.evict(0, d["big_w"], d["n"], keep + 50 * (i + 1), 4, 32, d["big_w"], d["n"], stream=stream)
        stream.synchronize()

    def results(d):
        return [d[k].to_host(np.uint32, d[k].nbytes // 4) for k in ("o", "o1", "o2", "w", "n")] + \
            [a for name in ("ring", "own") for a in read_rows(d[name].kv, 0)]

    stream = Stream()
    graphed, eager = state(), state()
    for d in (graphed, eager):
        feed(d, 2)
        step(d, stream)
        stream.synchronize()
    with Graph.capture(stream) as g:
        step(graphed, stream)
    for i in range(4):
        for d in (graphed, eager):
            feed(d, 10 + i)
        g.launch(stream)
        stream.synchronize()
        step(eager, stream)
        stream.synchronize()
        for a, b in zip(results(graphed), results(eager)):
            np.testing.assert_array_equal(a, b)
        for d in (graphed, eager):
            outgrow(d, stream, i)
    g.close()
