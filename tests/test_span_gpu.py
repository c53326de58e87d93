"""Attention over spans of the int8 cache (windows with pinned first positions, a shared prefix, recorded weights)
against the closed form in 64 bits, at the edges of its tiles, runs, row tiles and pieces.

Tolerance, per output. The products of codes and of the three bfloat16 terms of q are exact; a score's sum has at most
3 * head_dim rounded additions whose errors are independent, and four more roundings (its scale, that times the dot, the
maximum's subtraction, the exponential): e = (sqrt(3 * head_dim) + 4 * 4) * 2^-24 of its terms' magnitudes, in which the
last four count as worst cases of up to four units each. A weight is off by e times its score's magnitude, the sum of
weights by as much, and the value sum has sqrt(3 * keys) more: an output is off by at most
(2 * e * max_j sum_d |q_d K_jd| / sqrt(head_dim) + (sqrt(3 * keys) + 8) * 2^-24) * sum_j p_j |V_j|.
"""
import numpy as np
import pytest

import oracle
from openneedle_amd.device import DeviceArray, Graph, Stream, synchronize
from openneedle_amd.kv import KVCache
from tests.test_evict_gpu import kept_slots, read_rows, write_rows

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24


class Rows:
    """A layer's rows on the host, [seqs][slots][kvheads][head_dim] codes and scales, mirrored in a cache."""

    def __init__(self, rng, seqs, cap, kvh, hd, layers=1, layer=0):
        self.kv, self.layer = KVCache(layers, cap, kvh, hd, seqs), layer
        self.k, self.v = (rng.integers(-127, 128, (seqs, cap, kvh, hd)).astype(np.int8) for _ in "kv")
        self.ks, self.vs = (rng.uniform(0.01, 0.025, (seqs, cap, kvh)).astype(np.float32) for _ in "kv")
        self.push()

    def push(self):
        write_rows(self.kv, self.layer, (self.k, self.v, self.ks, self.vs))

    def put(self, s, slot, k, v):
        for codes, scales, rows in ((self.k, self.ks, k), (self.v, self.vs, v)):
            c, x = oracle.kv_quantize(rows[None])
            codes[s, slot], scales[s, slot] = c[0], x[0]

    def at(self, s, slots, h):
        slots = np.asarray(slots, np.int64)
        return ((self.k[s, slots, h].astype(np.float64) * self.ks[s, slots, h, None].astype(np.float64)),
                (self.v[s, slots, h].astype(np.float64) * self.vs[s, slots, h, None].astype(np.float64)))

    def same(self):
        """The cache holds exactly these rows."""
        for a, b in zip(read_rows(self.kv, self.layer), (self.k, self.v, self.ks, self.vs)):
            np.testing.assert_array_equal(a, b)


def attend(q, k, v):
    """(output, tolerance, weights) of one query row over rows k, v in 64 bits."""
    hd = q.shape[-1]
    if len(k) == 0:
        return np.zeros(hd), np.zeros(hd), np.zeros(0)
    q = q.astype(np.float64)
    x = k @ q / np.sqrt(hd)
    p = np.exp(x - x.max())
    p /= p.sum()
    e = (np.sqrt(3 * hd) + 16) * EPS
    size = (np.abs(k) @ np.abs(q)).max() / np.sqrt(hd)
    return p @ v, (2 * e * size + (np.sqrt(3 * len(k)) + 8) * EPS) * (p @ np.abs(v)) + 1e-37, p


def check(got, want, tol, what):
    bad = np.abs(got - want) > tol
    assert not bad.any(), f"{what}: off by {np.abs(got - want)[bad].max()} where {tol[bad].min()} is allowed"
    assert np.isfinite(got).all(), what


def ring_slot(p, sinks, cap):
    return p if p < sinks else sinks + (p - sinks) % (cap - sinks)


def seen(p, sinks, window):
    """Positions that a token at p attends."""
    return [] if p < 0 else [j for j in range(min(sinks, p + 1))] + list(range(max(sinks, p - window + 1), p + 1))


def upload(a, dtype=np.float32):
    return DeviceArray.from_host(np.asarray(a, dtype))


def run_window(r, q, positions, sinks, window, new=None, stream=None):
    out = DeviceArray.from_host(np.full(q.shape, np.nan, np.float32))
    d = [upload(q), upload(positions, np.int32)] + ([upload(n) for n in new] if new else [])
    r.kv.attention_window(r.layer, d[0], out, q.shape[2], q.shape[1], d[1], sinks, window, stream=stream,
                          new=tuple(d[2:]) if new else None)
    synchronize()
    return out.to_host(np.float32, q.shape)


def window_case(rng, kvh, group, hd, count, sinks, window, positions, extra=0, store=True, layers=1, layer=0):
    cap = sinks + window + count - 1 + extra
    seqs = len(positions)
    r = Rows(rng, seqs, cap, kvh, hd, layers, layer)
    q = rng.normal(size=(seqs, count, kvh * group, hd)).astype(np.float32)
    new = tuple(rng.normal(size=(seqs, count, kvh, hd)).astype(np.float32) for _ in "kv") if store else None
    got = run_window(r, q, positions, sinks, window, new)
    for s, first in enumerate(positions):
        for i in range(count):
            if store and first + i >= 0:
                r.put(s, ring_slot(first + i, sinks, cap), new[0][s, i], new[1][s, i])
    r.same()
    check_window(r, q, positions, sinks, window, got)


def check_window(r, q, positions, sinks, window, got, tokens=None):
    cap, kvh = r.k.shape[1], r.k.shape[2]
    group = q.shape[2] // kvh
    for s, first in enumerate(positions):
        for i in tokens if tokens is not None else range(q.shape[1]):
            slots = [ring_slot(j, sinks, cap) for j in seen(first + i, sinks, window)]
            for h in range(kvh):
                k, v = r.at(s, slots, h)
                for g in range(group):
                    want, tol, _ = attend(q[s, i, h * group + g], k, v)
                    check(got[s, i, h * group + g], want, tol, f"sequence {s} token {i} head {h * group + g}")


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("kvh,group", [(1, 1), (2, 2), (2, 3), (1, 8), (3, 5), (1, 16)])
def test_window_one_token(hd, kvh, group):
    """One token per sequence, before the window is full, around its edges and after many rounds; idle sequences."""
    rng = np.random.default_rng(hd + 10 * kvh + group)
    window_case(rng, kvh, group, hd, 1, 5, 64, [0, 4, 5, 63, 68, 69, 70, 131, 1000003, 2 ** 31 - 2, -1, -2 ** 31])
    window_case(rng, kvh, group, hd, 1, 0, 1, [0, 1, 77])
    window_case(rng, kvh, group, hd, 1, 3, 1, [0, 2, 3, 4], extra=2)


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("sinks,window,extra", [(0, 700, 0), (4, 700, 0), (4, 701, 130), (130, 600, 3)])
def test_window_several_pieces(hd, sinks, window, extra):
    """Few sequences over a long window: the keys are cut into pieces, some of them empty."""
    rng = np.random.default_rng(hd + window + extra)
    window_case(rng, 2, 4, hd, 1, sinks, window, [0, 200, window + sinks, 5 * window + 7, -1], extra=extra)


def test_window_long():
    rng = np.random.default_rng(77)
    window_case(rng, 1, 2, 64, 1, 16, 20000, [19999, 123456])
    window_case(rng, 1, 2, 128, 3, 16, 9001, [123456])


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("group,count", [(1, 2), (1, 17), (2, 8), (3, 5), (3, 6), (4, 33), (8, 3), (16, 2), (5, 64), (1, 130)])
def test_window_several_tokens(hd, group, count):
    """Drafts and prompt pieces: rows of several tokens in one tile, left padding, window shorter and longer than the
    piece, wraps inside it."""
    rng = np.random.default_rng(hd + 100 * group + count)
    window_case(rng, 2, group, hd, count, 3, 40, [0, -count, 1 - count, -2, 41, 45, 12345])
    window_case(rng, 1, group, hd, count, 0, 150, [149, 2, 700], extra=1)
    window_case(rng, 1, group, hd, count, 70, 1, [0, 69, 500], extra=64)


@pytest.mark.parametrize("group,count,window", [(2, 300, 100), (4, 257, 500), (1, 513, 65)])
def test_window_prompt_pieces(group, count, window):
    rng = np.random.default_rng(count)
    window_case(rng, 2, group, 64, count, 4, window, [0, 1000])


def test_window_rows_stored_before():
    """Without new rows the tokens' own rows are taken from the cache; the second of two layers."""
    rng = np.random.default_rng(5)
    window_case(rng, 2, 2, 64, 1, 4, 100, [0, 99, 500], store=False, layers=2, layer=1)
    window_case(rng, 2, 2, 64, 9, 4, 100, [0, 99, 500], store=False, layers=2, layer=1)


@pytest.mark.parametrize("count", [1, 4, 40])
def test_window_what_is_not_attended_does_not_matter(count):
    """Slots outside the window hold infinite and NaN scales."""
    rng = np.random.default_rng(6)
    sinks, window, hd = 4, 50, 64
    cap = sinks + window + count - 1 + 90
    r = Rows(rng, 3, cap, 2, hd)
    positions = [20, 300, 501]
    for s, first in enumerate(positions):
        live = {ring_slot(j, sinks, cap) for i in range(count) for j in seen(first + i, sinks, window)}
        dead = [j for j in range(cap) if j not in live]
        assert dead
        r.ks[s, dead[::2]] = np.nan
        r.ks[s, dead[1::2]] = np.inf
        r.vs[s, dead[::3]] = np.inf
        r.vs[s, dead[1::3]] = np.nan
    r.push()
    q = rng.normal(size=(3, count, 4, hd)).astype(np.float32)
    check_window(r, q, positions, sinks, window, run_window(r, q, positions, sinks, window))


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("ratio", [1e4, 1e8, 1e30])
def test_uneven_queries_and_weights(hd, ratio):
    """An entry of q far above the rest over zero K codes; a slot far ahead with zero V codes in half of its
    dimensions: the other terms keep their own precision."""
    rng = np.random.default_rng(int(np.log10(ratio)) + hd)
    r = Rows(rng, 1, 300, 2, hd)
    r.k[0, :, :, 5] = 0
    r.v[0, 77, :, ::2] = 0
    r.v[0, :, :, ::2] = np.abs(r.v[0, :, :, ::2])
    q = rng.normal(size=(1, 1, 4, hd)).astype(np.float32)
    r.k[0, 77] = np.where(q[0, 0, ::2] > 0, 127, -127)
    r.k[0, :, :, 5] = 0
    r.ks[0, 77] = 0.05
    q[..., 5] = ratio
    r.push()
    check_window(r, q, [299], 0, 300, run_window(r, q, [299], 0, 300))


def test_non_finite_input():
    """A head with an infinity or NaN in its query has no softmax and yields zeros, the others are untouched; an
    infinite V scale gives infinities of the codes' signs (NaN for a zero code) to its kv head alone."""
    rng = np.random.default_rng(8)
    for count in (1, 20):
        r = Rows(rng, 1, 400, 2, 64)
        q = rng.normal(size=(1, count, 8, 64)).astype(np.float32)
        q[0, 0, 0, 3] = np.nan
        q[0, 0, 2, 9] = np.inf
        got = run_window(r, q, [399 - count + 1], 0, 380)
        assert not got[0, 0, [0, 2]].any()
        q[0, 0, [0, 2]] = 0
        keep = got.copy()
        keep[0, 0, [0, 2]] = run_window(r, q, [399 - count + 1], 0, 380)[0, 0, [0, 2]]
        check_window(r, q, [399 - count + 1], 0, 380, keep)
        r.vs[0, 200, 1] = np.inf
        r.v[0, 200, 1, 3] = 0
        r.push()
        got = run_window(r, q, [399 - count + 1], 0, 380)
        assert np.isfinite(got[:, :, :4]).all()
        codes = r.v[0, 200, 1]
        want = np.where(codes == 0, np.nan, np.where(codes > 0, np.inf, -np.inf))
        for h in range(4, 8):
            np.testing.assert_array_equal(got[0, 0, h], want)


# ---- many rows over the same keys: two float16 terms ----------------------------------------------------------------
def check_many_rows(r, q, first, got):
    """A prompt piece over a window of first + 1 positions, the first token's from position 0 on (slot = position, tiles of
    32 slots): the tolerance above, whose sums have room for the terms' 2^-22 per value and 2^-24 per score, plus what the terms of a weight leave: at most
    2^-27 of the largest p * v_scale among the tile's 32."""
    kvh, hd = r.k.shape[2], q.shape[-1]
    group = q.shape[2] // kvh
    for i in range(q.shape[1]):
        at = np.arange(i, first + i + 1)
        for h in range(kvh):
            k, v = r.at(0, at, h)
            vs, codes = np.abs(r.vs[0, at, h].astype(np.float64)), np.abs(r.v[0, at, h].astype(np.float64))
            for g in range(group):
                want, tol, p = attend(q[0, i, h * group + g], k, v)
                for t in np.unique(at // 32):
                    mine = at // 32 == t
                    tol = tol + 2.0 ** -27 * (p[mine] * vs[mine]).max() * codes[mine].sum(0)
                check(got[0, i, h * group + g], want, tol, f"token {i} head {h * group + g}")


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("ratio", [1e4, 1e6, 1e8, 1e12, 1e30])
def test_many_rows_uneven_queries(hd, ratio):
    """Entries of q far above the rest over zero K codes, in some rows only: the other entries' products decide."""
    rng = np.random.default_rng(hd + int(np.log10(ratio)))
    r = Rows(rng, 1, 340, 2, hd)
    r.k[:, :, :, 5] = 0
    r.push()
    q = rng.normal(size=(1, 40, 4, hd)).astype(np.float32)
    q[0, 3::7, :, 5] = ratio
    q[0, 5] *= 1e-30
    q[0, 6] = 0
    check_many_rows(r, q, 300, run_window(r, q, [300], 0, 301))


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("margin", [3, 10, 30, 60, 120])
def test_many_rows_dominant_slots(hd, margin):
    """Some slots whose scores are `margin` above the rest, with zero V codes in half of the dimensions: there the other
    slots' sums show, down to e^-120 of the weights (the smallest normal number is e^-87: less is lost, within 1e-37)."""
    rng = np.random.default_rng(hd + margin)
    r = Rows(rng, 1, 340, 2, hd)
    sign = rng.choice([-1, 1], hd)
    q = (np.abs(rng.normal(size=(1, 40, 4, hd))) * sign).astype(np.float32)
    for j in (0, 77, 200):
        r.k[0, j] = 127 * sign
        r.ks[0, j] = margin * np.sqrt(hd) / (127 * np.abs(q).sum(-1).mean())
        r.v[0, j, :, ::2] = 0
    r.push()
    check_many_rows(r, q, 300, run_window(r, q, [300], 0, 301))


@pytest.mark.parametrize("scales", ["tiny", "huge", "mixed", "zero", "signed"])
def test_many_rows_v_scales(scales):
    rng = np.random.default_rng(50)
    r = Rows(rng, 1, 340, 2, 64)
    if scales == "tiny":
        r.vs *= np.float32(2.0 ** -108)
    elif scales == "huge":
        r.vs *= np.float32(2.0 ** 118)
    elif scales == "mixed":
        r.vs[0, :160] *= np.float32(2.0 ** -100)
        r.vs[0, 100] = 2.0 ** 90
        r.vs[0, 200:] *= np.float32(2.0 ** -30)
    elif scales == "zero":
        r.vs[0, :200] = 0
    else:
        r.vs[0, ::3] *= -1
        r.ks[0, ::2] *= -1
    r.push()
    q = rng.normal(size=(1, 40, 4, 64)).astype(np.float32)
    check_many_rows(r, q, 300, run_window(r, q, [300], 0, 301))


# ---- a shared prefix ----------------------------------------------------------------------------------------------
def run_shared(r, prefix, prefix_length, q, length, lengths, new=None, prefix_seq=0, stream=None):
    out = DeviceArray.from_host(np.full(q.shape, np.nan, np.float32))
    d = [upload(q), upload(lengths, np.int32) if lengths is not None else None] + ([upload(n) for n in new] if new else [])
    r.kv.attention_shared(r.layer, prefix.kv, prefix_length, d[0], out, q.shape[1], length, d[1], prefix_seq=prefix_seq,
                          stream=stream, new=tuple(d[2:]) if new else None)
    synchronize()
    return out.to_host(np.float32, q.shape)


def check_shared(r, prefix, prefix_length, prefix_seq, q, lengths, got):
    kvh = r.k.shape[2]
    group = q.shape[1] // kvh
    for h in range(kvh):
        pk, pv = prefix.at(prefix_seq, range(prefix_length), h)
        for s, n in enumerate(lengths):
            k, v = r.at(s, range(max(n, 0)), h)
            k, v = np.concatenate([pk, k]), np.concatenate([pv, v])
            for g in range(group):
                want, tol, _ = attend(q[s, h * group + g], k, v)
                check(got[s, h * group + g], want, tol, f"sequence {s} head {h * group + g}")


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("seqs,kvh,group", [(1, 1, 1), (3, 2, 2), (5, 1, 8), (17, 2, 3), (40, 1, 4), (2, 1, 16), (70, 2, 4)])
@pytest.mark.parametrize("prefix_length", [0, 1, 64, 65, 700])
def test_shared_prefix(hd, seqs, kvh, group, prefix_length):
    rng = np.random.default_rng(hd + seqs + 31 * prefix_length)
    prefix = Rows(rng, 2, 701, kvh, hd, layers=2, layer=1)
    r = Rows(rng, seqs, 150, kvh, hd, layers=2, layer=1)
    lengths = rng.integers(0, 150, seqs)
    lengths[0] = 149
    lengths[-1] = 1 if seqs == 1 else 0
    q = rng.normal(size=(seqs, kvh * group, hd)).astype(np.float32)
    new = tuple(rng.normal(size=(seqs, kvh, hd)).astype(np.float32) for _ in "kv")
    got = run_shared(r, prefix, prefix_length, q, 149, lengths, new, prefix_seq=1)
    for s, n in enumerate(lengths):
        if n > 0:
            r.put(s, n - 1, new[0][s], new[1][s])
    r.same()
    prefix.same()
    check_shared(r, prefix, prefix_length, 1, q, lengths, got)


def test_shared_prefix_long_and_short():
    """A prefix of many pieces; sequences without any slot of their own; lengths beyond `length` and below zero."""
    rng = np.random.default_rng(3)
    prefix = Rows(rng, 1, 30011, 2, 64)
    r = Rows(rng, 9, 64, 2, 64)
    q = rng.normal(size=(9, 8, 64)).astype(np.float32)
    got = run_shared(r, prefix, 30011, q, 0, None)
    check_shared(r, prefix, 30011, 0, q, [0] * 9, got)
    got = run_shared(r, prefix, 100, q, 33, [200, -3, 0, 1, 33, 34, 32, 2, 2 ** 31 - 1])
    check_shared(r, prefix, 100, 0, q, [33, 0, 0, 1, 33, 33, 32, 2, 33], got)
    got = run_shared(r, prefix, 0, q, 33, [200, -3, 0, 1, 33, 34, 32, 2, 5])  # nothing at all for two of them
    check_shared(r, prefix, 0, 0, q, [33, 0, 0, 1, 33, 33, 32, 2, 5], got)


def test_shared_prefix_equals_the_same_rows_in_one_cache():
    """The prefix copied in front of every sequence's own rows, through `attention`: the same up to both tolerances."""
    rng = np.random.default_rng(4)
    prefix, r = Rows(rng, 1, 200, 2, 64), Rows(rng, 4, 60, 2, 64)
    both = Rows(rng, 4, 260, 2, 64)
    for s in range(4):
        for name in ("k", "v", "ks", "vs"):
            getattr(both, name)[s] = np.concatenate([getattr(prefix, name)[0], getattr(r, name)[s]])
    both.push()
    q = rng.normal(size=(4, 4, 64)).astype(np.float32)
    got = run_shared(r, prefix, 200, q, 60, None)
    d_q, d_o = upload(q), DeviceArray(q.nbytes)
    both.kv.attention(0, d_q, d_o, 4, 260)
    synchronize()
    np.testing.assert_allclose(got, d_o.to_host(np.float32, q.shape), atol=2e-6, rtol=2e-5)


# ---- recorded weights -----------------------------------------------------------------------------------------------
def run_weights(r, q, record, length, lengths, new=None, stream=None):
    out = DeviceArray.from_host(np.full(q.shape, np.nan, np.float32))
    d_w = upload(record)
    d = [upload(q), upload(lengths, np.int32) if lengths is not None else None] + ([upload(n) for n in new] if new else [])
    r.kv.attention_weights(r.layer, d[0], out, d_w, q.shape[1], length, d[1], stream=stream, new=tuple(d[2:]) if new else None)
    synchronize()
    return out.to_host(np.float32, q.shape), d_w.to_host(np.float32, record.shape)


def check_weights(r, q, record, lengths, got, got_w):
    kvh = r.k.shape[2]
    group = q.shape[1] // kvh
    hd = q.shape[-1]
    for s, n in enumerate(lengths):
        for h in range(kvh):
            k, v = r.at(s, range(n), h)
            add, tol_w = np.zeros(n), np.zeros(n)
            for g in range(group):
                row = q[s, h * group + g]
                if not np.isfinite(row).all():
                    assert not got[s, h * group + g].any()
                    continue
                want, tol, p = attend(row, k, v)
                check(got[s, h * group + g], want, tol, f"sequence {s} head {h * group + g}")
                add += p
                if n:
                    e = (np.sqrt(3 * hd) + 16) * EPS * (np.abs(k) @ np.abs(row.astype(np.float64))).max() / np.sqrt(hd)
                    tol_w += (2 * e + (np.sqrt(n) + 8) * EPS) * p
            # the record's own addition and the sum over the group round once each
            want = record[s, h, :n].astype(np.float64) + add
            tol_w += EPS * (np.abs(want) + (group + 1) * add)
            assert (np.abs(got_w[s, h, :n] - want) <= tol_w + 1e-37).all(), f"sequence {s} kv head {h}"
            np.testing.assert_array_equal(got_w[s, h, n:], record[s, h, n:])


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("kvh,group", [(1, 1), (2, 3), (3, 8), (1, 16)])
@pytest.mark.parametrize("length", [1, 64, 65, 300, 1500])
def test_weights(hd, kvh, group, length):
    rng = np.random.default_rng(hd + group + length)
    seqs, cap = 4, length + 3
    r = Rows(rng, seqs, cap, kvh, hd, layers=2, layer=1)
    lengths = [length, max(1, length // 2), 0, max(1, length - 1)]
    q = rng.normal(size=(seqs, kvh * group, hd)).astype(np.float32)
    new = tuple(rng.normal(size=(seqs, kvh, hd)).astype(np.float32) for _ in "kv")
    record = rng.uniform(0, 3, (seqs, kvh, cap)).astype(np.float32)
    record[:, :, length:] = np.nan  # not the call's
    got, got_w = run_weights(r, q, record, length, lengths, new)
    for s, n in enumerate(lengths):
        if n:
            r.put(s, n - 1, new[0][s], new[1][s])
    r.same()
    check_weights(r, q, record, lengths, got, got_w)


def test_weights_without_a_softmax_and_to_capacity():
    rng = np.random.default_rng(12)
    r = Rows(rng, 2, 333, 2, 64)
    q = rng.normal(size=(2, 6, 64)).astype(np.float32)
    q[0, 1, 7] = np.nan
    q[1, 5, 0] = -np.inf
    record = np.zeros((2, 2, 333), np.float32)
    got, got_w = run_weights(r, q, record, 333, None)
    check_weights(r, q, record, [333, 333], got, got_w)
    # every head with a softmax gave the kv head's slots a whole weight
    np.testing.assert_allclose(got_w.sum(-1, dtype=np.float64), [[2, 3], [3, 2]], rtol=(np.sqrt(333) + 30) * 2 * EPS)


# ---- together -------------------------------------------------------------------------------------------------------
def test_decode_record_evict_and_go_on():
    """A batch decodes with its weights recorded, is cut by the record, and goes on: every step's outputs, the record
    and the kept slots against the same steps in 64 bits."""
    rng = np.random.default_rng(20)
    seqs, kvh, group, hd, cap, keep = 3, 2, 4, 64, 320, 150
    r = Rows(rng, seqs, cap, kvh, hd)
    lengths = np.array([310, 200, 120], np.int32)
    record = np.zeros((seqs, kvh, cap), np.float32)
    d_w, d_n = upload(record), upload(lengths, np.int32)
    d_q, d_k, d_v = (DeviceArray(seqs * n * hd * 4) for n in (kvh * group, kvh, kvh))
    d_o = DeviceArray(seqs * kvh * group * hd * 4)
    stream = Stream()
    for step in range(6):
        lengths += 1
        d_n.upload(lengths)
        q = rng.normal(size=(seqs, kvh * group, hd)).astype(np.float32)
        new = tuple(rng.normal(size=(seqs, kvh, hd)).astype(np.float32) for _ in "kv")
        for d, a in zip((d_q, d_k, d_v), (q, *new)):
            d.upload(a)
        before = d_w.to_host(np.float32, record.shape)
        r.kv.attention_weights(0, d_q, d_o, d_w, kvh * group, cap, d_n, stream=stream, new=(d_k, d_v))
        stream.synchronize()
        for s, n in enumerate(lengths):
            r.put(s, n - 1, new[0][s], new[1][s])
        after = d_w.to_host(np.float32, record.shape)
        check_weights(r, q, before, lengths, d_o.to_host(np.float32, q.shape), after)
        if step in (2, 4):
            r.kv.evict(0, d_w, d_n, keep, 4, 30, d_w, d_n, stream=stream)
            stream.synchronize()
            cut = d_w.to_host(np.float32, record.shape)
            for s, n in enumerate(lengths):
                for h in range(kvh):
                    slots = kept_slots(after[s, h], n, keep, 4, 30)
                    for a in (r.k, r.v, r.ks, r.vs):
                        a[s, :len(slots), h] = a[s, slots, h]
                    np.testing.assert_array_equal(cut[s, h, :len(slots)], after[s, h, slots])
                    assert not cut[s, h, len(slots):].any()
            lengths = np.minimum(lengths, keep).astype(np.int32)
            np.testing.assert_array_equal(d_n.to_host(np.int32, seqs), lengths)
            r.same()


@pytest.mark.parametrize("count", [1, 6])
def test_graph_replays_match_eager(count):
    """A window step, a shared-prefix step, a recorded step and a cut captured into one graph, replayed with other
    inputs and eager calls of larger sizes in between (whose scratch must not move the graph's)."""
    seqs, kvh, heads, hd, sinks, window = 2, 2, 8, 64, 4, 600
    cap = sinks + window + count - 1

    def state(seed):
        rng = np.random.default_rng(seed)
        d = dict(ring=Rows(rng, seqs, cap, kvh, hd), own=Rows(rng, seqs, 400, kvh, hd), prefix=Rows(rng, 1, 900, kvh, hd))
        d["q"], d["nk"], d["nv"], d["o"] = (DeviceArray(seqs * count * n * hd * 4) for n in (heads, kvh, kvh, heads))
        d["q1"], d["k1"], d["v1"], d["o1"], d["o2"] = (DeviceArray(seqs * n * hd * 4) for n in (heads, kvh, kvh, heads, heads))
        d["pos"], d["n"], d["n2"] = (DeviceArray(seqs * 4) for _ in range(3))
        d["w"], d["w2"] = DeviceArray(seqs * kvh * 400 * 4), DeviceArray(seqs * kvh * 400 * 4)
        return d

    def feed(d, seed):
        rng = np.random.default_rng(seed)
        for name in ("q", "nk", "nv", "q1", "k1", "v1"):
            d[name].upload(rng.normal(size=d[name].nbytes // 4).astype(np.float32))
        d["pos"].upload(rng.integers(0, 3000, seqs).astype(np.int32))
        d["n"].upload(rng.integers(200, 400, seqs).astype(np.int32))
        d["w"].upload(rng.random(seqs * kvh * 400).astype(np.float32))

    def step(d, stream):
        d["ring"].kv.attention_window(0, d["q"], d["o"], heads, count, d["pos"], sinks, window, stream=stream,
                                      new=(d["nk"], d["nv"]))
        d["own"].kv.attention_shared(0, d["prefix"].kv, 900, d["q1"], d["o1"], heads, 400, d["n"], stream=stream,
                                     new=(d["k1"], d["v1"]))
        d["own"].kv.attention_weights(0, d["q1"], d["o2"], d["w"], heads, 400, d["n"], stream=stream)
        d["own"].kv.evict(0, d["w"], d["n"], 128, 4, 32, d["w2"], d["n2"], stream=stream)

    def results(d):
        return [d[k].to_host(np.uint32, d[k].nbytes // 4) for k in ("o", "o1", "o2", "w", "w2", "n2")] + \
            [a for name in ("ring", "own") for a in read_rows(d[name].kv, 0)]

    stream = Stream()
    graphed, eager = state(1), state(1)
    feed(graphed, 2)
    feed(eager, 2)
    step(graphed, stream)
    stream.synchronize()
    step(eager, stream)
    stream.synchronize()
    with Graph.capture(stream) as g:
        step(graphed, stream)
    more = DeviceArray(seqs * 32 * hd * 4)
    for i in range(4):
        feed(graphed, 10 + i)
        feed(eager, 10 + i)
        g.launch(stream)
        stream.synchronize()
        step(eager, stream)
        stream.synchronize()
        for a, b in zip(results(graphed), results(eager)):
            np.testing.assert_array_equal(a, b)
        # more heads than the captured calls: larger scratch of the same handles
        more.fill(0)
        d_w = DeviceArray(seqs * kvh * 400 * 4)
        d_w.fill(0)
        graphed["own"].kv.attention_weights(0, more, more, d_w, 32, 400, graphed["n"], stream=stream)
        stream.synchronize()
    g.close()


def test_unaligned_buffers_and_growing_lengths():
    """Buffers that start at any float; a length that grows with every step (the scratch does not grow with it)."""
    rng = np.random.default_rng(33)
    r = Rows(rng, 2, 300, 2, 64)
    q = rng.normal(size=(2, 4, 64)).astype(np.float32)
    record = np.zeros((2, 2, 300), np.float32)
    big = [DeviceArray(n + 16) for n in (q.nbytes, q.nbytes, record.nbytes, q.nbytes // 2, q.nbytes // 2)]
    for off in (4, 8, 12):
        d_q, d_o, d_w, d_k, d_v = (b.view(off, b.nbytes - 16) for b in big)
        for length in range(10, 301, 29):
            new = tuple(rng.normal(size=(2, 2, 64)).astype(np.float32) for _ in "kv")
            for d, a in zip((d_q, d_w, d_k, d_v), (q, record, *new)):
                d.upload(a)
            r.kv.attention_weights(0, d_q, d_o, d_w, 4, length, new=(d_k, d_v))
            synchronize()
            for s in range(2):
                r.put(s, length - 1, new[0][s], new[1][s])
            got_w = d_w.to_host(np.float32, record.shape)
            check_weights(r, q, record, [length] * 2, d_o.to_host(np.float32, q.shape), got_w)
        d_n = upload([299, 299], np.int32)
        many, d_m = rng.normal(size=(2, 40, 4, 64)).astype(np.float32), DeviceArray(2 * 40 * 4 * 64 * 4 + 16)
        d_p, d_r = d_m.view(off, d_m.nbytes - 16), DeviceArray(d_m.nbytes)
        d_p.upload(many)
        d_r = d_r.view(off, d_m.nbytes - 16)
        r.kv.attention_window(0, d_p, d_r, 4, 40, d_n, 4, 200)
        synchronize()
        check_window(r, many, [299, 299], 4, 200, d_r.to_host(np.float32, many.shape), tokens=(0, 17, 39))
    r.same()


def test_same_results_every_time():
    rng = np.random.default_rng(30)
    r = Rows(rng, 2, 3000, 2, 128)
    q = rng.normal(size=(2, 1, 8, 128)).astype(np.float32)
    first = run_window(r, q, [2999, 10000], 0, 3000)
    for _ in range(3):
        np.testing.assert_array_equal(run_window(r, q, [2999, 10000], 0, 3000), first)


def test_refusals_change_nothing():
    rng = np.random.default_rng(40)
    r, p = Rows(rng, 2, 32, 2, 64), Rows(rng, 1, 16, 2, 64)
    other = KVCache(1, 16, 2, 32, 1)
    d, i = DeviceArray(2 * 2 * 40 * 64 * 4), upload([31, 31], np.int32)
    d.fill(0)
    kv = r.kv
    for args, word in [((0, d, d, 3, 1, i, 4, 16), "multiple"), ((0, d, d, 34, 1, i, 4, 16), "16 query heads"),
                       ((0, d, d, 4, 1, i, 17, 16), "capacity"), ((0, d, d, 4, 14, i, 4, 16), "capacity"),
                       ((0, d, d, 4, 1, i, 4, 0), "window"), ((0, d, d, 4, 1, i, -1, 4), "sinks"),
                       ((0, d, d, 4, -1, i, 4, 16), "count"), ((1, d, d, 4, 1, i, 4, 16), "layer"),
                       ((0, None, d, 4, 1, i, 4, 16), "null"), ((0, d, d, 4, 1, None, 4, 16), "null")]:
        with pytest.raises(RuntimeError, match=word):
            kv.attention_window(*args, new=(d, d))
    with pytest.raises(RuntimeError, match="come together"):
        kv.attention_window(0, d, d, 4, 1, i, 4, 16, new=(d, None))
    for args, word in [((0, p.kv, 17, d, d, 4, 32), "prefix length"), ((0, p.kv, 16, d, d, 4, 33), "length"),
                       ((0, other, 16, d, d, 4, 32), "geometry"), ((0, kv, 16, d, d, 4, 32), "cache of its own"),
                       ((0, p.kv, 16, None, d, 4, 32), "null"), ((0, p.kv, 16, d, d, 5, 32), "multiple")]:
        with pytest.raises(RuntimeError, match=word):
            kv.attention_shared(*args, new=(d, d))
    with pytest.raises(RuntimeError, match="prefix sequence"):
        kv.attention_shared(0, p.kv, 16, d, d, 4, 32, prefix_seq=1)
    for args, word in [((0, d, d, None, 4, 32), "null"), ((0, d, d, d, 4, 33), "length"), ((0, d, d, d, 4, -1), "length"),
                       ((0, d, d, d, 6 * 17, 32), "16 query heads")]:
        with pytest.raises(RuntimeError, match=word):
            kv.attention_weights(*args, new=(d, d))
    kv.attention_window(0, d, d, 4, 0, i, 4, 16)  # no tokens: nothing to do
    synchronize()
    r.same()
    p.same()


def test_device_rows():
    rng = np.random.default_rng(41)
    r = Rows(rng, 2, 9, 3, 32, layers=2, layer=1)
    for s in range(2):  # written through device_rows, read as host rows
        for a, b in zip(r.kv.read(1, s, 9), (r.k, r.v, r.ks, r.vs)):
            np.testing.assert_array_equal(a, b[s])
        r.kv.load(1, s, r.k[1 - s], r.v[1 - s], r.ks[1 - s], r.vs[1 - s])
    for a, b in zip(read_rows(r.kv, 1), (r.k, r.v, r.ks, r.vs)):
        np.testing.assert_array_equal(a, b[::-1])
    with pytest.raises(RuntimeError, match="layer"):
        r.kv.device_rows(2)
