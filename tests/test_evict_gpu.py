"""Eviction of the int8 cache by recorded weights: kept slots, rows, scales, weights and lengths exactly as a plain
stable sort gives them."""
import numpy as np
import pytest

from openneedle_amd.device import DeviceArray, Stream, synchronize
from openneedle_amd.kv import KVCache


def kept_slots(w, n, keep, sinks, recent):
    """Slots that a (sequence, kv head) with weights w keeps of its first n, in order."""
    if n <= keep:
        return list(range(n))
    middle = np.asarray(w[sinks:n - recent], np.float64)
    rank = np.where(np.isnan(middle), -np.inf, middle)
    order = np.lexsort((np.arange(len(rank)), np.isnan(middle), -rank))[:keep - sinks - recent]
    return sorted([*range(sinks), *(order + sinks).tolist(), *range(n - recent, n)])


def filled(rng, seqs, cap, kvh, hd, layers=1):
    """A cache of random codes and scales, and its rows per (layer, sequence)."""
    kv = KVCache(layers, cap, kvh, hd, seqs)
    rows = {}
    for layer in range(layers):
        for s in range(seqs):
            k, v = (rng.integers(-127, 128, (cap, kvh, hd)).astype(np.int8) for _ in "kv")
            ks, vs = (rng.uniform(0.01, 0.03, (cap, kvh)).astype(np.float32) for _ in "kv")
            rows[layer, s] = (k, v, ks, vs)
        write_rows(kv, layer, [np.stack([rows[layer, s][i] for s in range(seqs)]) for i in range(4)])
    return kv, rows


def write_rows(kv, layer, rows):
    """(k, v, ks, vs) [seqs][slots][kvheads]... of a whole layer into the cache, through its device memory."""
    for at, a in zip(kv.device_rows(layer), rows):
        at.upload(np.swapaxes(a, 1, 2))


def read_rows(kv, layer):
    """The same back."""
    shape = (kv.seqs, kv.kvheads, kv.capacity)
    shapes = (shape + (kv.head_dim,),) * 2 + (shape,) * 2
    kinds = (np.int8, np.int8, np.float32, np.float32)
    return [np.swapaxes(at.to_host(k, n), 1, 2) for at, k, n in zip(kv.device_rows(layer), kinds, shapes)]


def run(kv, w, lengths, keep, sinks, recent, layer=0, alias=False, kept=True, stream=None):
    """(weights, lengths, kept) after the call, from device buffers (the weights' and lengths' own where `alias`)."""
    d_w, d_n = DeviceArray.from_host(w), DeviceArray.from_host(np.asarray(lengths, np.int32))
    d_w2 = d_w if alias else DeviceArray.from_host(np.full(w.shape, 7, np.float32))
    d_n2 = d_n if alias else DeviceArray.from_host(np.full(len(lengths), 7, np.int32))
    d_k = DeviceArray.from_host(np.full((kv.seqs, kv.kvheads, keep), 7, np.int32)) if kept else None
    kv.evict(layer, d_w, d_n, keep, sinks, recent, d_w2, d_n2, d_k, stream=stream)
    synchronize()
    if not alias:  # the inputs stay as they were
        np.testing.assert_array_equal(d_w.to_host(np.float32, w.shape), w)
        np.testing.assert_array_equal(d_n.to_host(np.int32, len(lengths)), lengths)
    return (d_w2.to_host(np.float32, w.shape), d_n2.to_host(np.int32, len(lengths)),
            d_k.to_host(np.int32, (kv.seqs, kv.kvheads, keep)) if kept else None)


def check(kv, rows, w, lengths, keep, sinks, recent, got, layer=0):
    new_w, new_n, kept = got
    cap = kv.capacity
    now = read_rows(kv, layer)
    for s in range(kv.seqs):
        n = min(max(int(lengths[s]), 0), cap)
        left = min(n, keep)
        assert new_n[s] == left
        after = [a.copy() for a in rows[layer, s]]
        for h in range(kv.kvheads):
            slots = kept_slots(w[s, h], n, keep, sinks, recent)
            assert len(slots) == left
            if kept is not None:
                np.testing.assert_array_equal(kept[s, h], slots + [-1] * (keep - left))
            np.testing.assert_array_equal(new_w[s, h], np.concatenate([w[s, h, slots], np.zeros(cap - left, np.float32)]))
            for a, b in zip(after, rows[layer, s]):
                a[:left, h] = b[slots, h]
        for a, b in zip(now, after):
            np.testing.assert_array_equal(a[s], b, err_msg=f"sequence {s}")


def weights(rng, seqs, kvh, cap):
    w = np.exp(2 * rng.normal(size=(seqs, kvh, cap)) - 4).astype(np.float32)
    w[rng.random(w.shape) < 0.1] = 0
    return w


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("cap,keep,sinks,recent,lengths", [
    (40, 16, 2, 5, [40, 17, 16]), (40, 16, 2, 5, [0, 3, 1000]), (40, 40, 0, 0, [40, 39, -5]), (1, 1, 0, 0, [1, 0, 1]),
    (65, 1, 0, 0, [65, 2, 1]), (65, 1, 1, 0, [65, 64, 2]), (65, 1, 0, 1, [65, 64, 2]), (300, 64, 32, 32, [300, 64, 65]),
    (1027, 511, 4, 100, [1027, 700, 512]), (5003, 2500, 0, 0, [5003, 4097, 4096]), (5003, 4999, 3, 17, [5003, 5000, 4999])])
def test_against_a_sort(hd, cap, keep, sinks, recent, lengths):
    rng = np.random.default_rng(cap * 7 + keep + hd)
    kv, rows = filled(rng, 3, cap, 2, hd)
    w = weights(rng, 3, 2, cap)
    check(kv, rows, w, lengths, keep, sinks, recent, run(kv, w, lengths, keep, sinks, recent))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["equal", "two", "zeros", "negative", "odd"])
def test_ties_and_odd_weights(kind):
    rng = np.random.default_rng(5)
    seqs, kvh, cap, hd = 2, 3, 4500, 32
    kv, rows = filled(rng, seqs, cap, kvh, hd)
    w = weights(rng, seqs, kvh, cap)
    if kind == "equal":
        w[:] = 0.25
    elif kind == "two":
        w = rng.choice([1.0, np.nextafter(np.float32(1), np.float32(2))], w.shape).astype(np.float32)
    elif kind == "zeros":
        w = np.where(rng.random(w.shape) < 0.5, np.float32(0.0), np.float32(-0.0))
    elif kind == "negative":
        w = rng.normal(size=w.shape).astype(np.float32)
    else:
        w[rng.random(w.shape) < 0.3] = np.nan
        w[rng.random(w.shape) < 0.3] = np.inf
        w[rng.random(w.shape) < 0.1] = -np.inf
        w[rng.random(w.shape) < 0.1] = 1e-42
    for keep, sinks, recent in [(2000, 10, 20), (4400, 0, 1), (9, 4, 4)]:
        kv, rows = filled(rng, seqs, cap, kvh, hd)
        lengths = [cap, cap - 3]
        got = run(kv, w, lengths, keep, sinks, recent)
        # a NaN weight that is kept moves as it is; -inf and NaN differ in rank only
        check(kv, rows, w, lengths, keep, sinks, recent, got)


@pytest.mark.gpu
@pytest.mark.parametrize("kept", [True, False])
def test_in_place_layers_and_streams(kept):
    """Weights and lengths updated in place, the second of three layers only, on a stream of its own."""
    rng = np.random.default_rng(9)
    cap, hd = 700, 64
    kv, rows = filled(rng, 2, cap, 2, hd, layers=3)
    w = weights(rng, 2, 2, cap)
    stream = Stream()
    got = run(kv, w, [700, 650], 333, 4, 32, layer=1, alias=True, kept=kept, stream=stream)
    check(kv, rows, w, [700, 650], 333, 4, 32, got, layer=1)
    for layer in (0, 2):
        for i, a in enumerate(read_rows(kv, layer)):
            for s in range(2):
                np.testing.assert_array_equal(a[s], rows[layer, s][i])


@pytest.mark.gpu
def test_many_sequences_and_a_second_cut():
    """A batch of more blocks than compute units, cut twice: the second cut keeps the first's oldest and newest."""
    rng = np.random.default_rng(10)
    seqs, kvh, cap, hd = 70, 4, 600, 128
    kv, rows = filled(rng, seqs, cap, kvh, hd)
    w = weights(rng, seqs, kvh, cap)
    lengths = rng.integers(0, cap + 1, seqs).astype(np.int32)
    got = run(kv, w, lengths, 257, 4, 30)
    check(kv, rows, w, lengths, 257, 4, 30, got)
    now = read_rows(kv, 0)
    rows = {(0, s): tuple(a[s] for a in now) for s in range(seqs)}
    again = run(kv, got[0], got[1], 100, 4, 30)
    check(kv, rows, got[0], got[1], 100, 4, 30, again)


@pytest.mark.gpu
def test_refusals_change_nothing():
    rng = np.random.default_rng(11)
    kv, rows = filled(rng, 1, 32, 2, 64)
    d_w, d_n = DeviceArray.from_host(weights(rng, 1, 2, 32)), DeviceArray.from_host(np.array([32], np.int32))
    for keep, sinks, recent, layer, word in [(0, 0, 0, 0, "keep"), (33, 0, 0, 0, "capacity"), (8, 5, 4, 0, "exceeds keep"),
                                             (8, -1, 4, 0, ">= 0"), (8, 1, -4, 0, ">= 0"), (8, 1, 4, 1, "layer")]:
        with pytest.raises(RuntimeError, match=word):
            kv.evict(layer, d_w, d_n, keep, sinks, recent, d_w, d_n)
    with pytest.raises(RuntimeError, match="null"):
        kv.evict(0, None, d_n, 8, 1, 4, d_w, d_n)
    with pytest.raises(RuntimeError, match="null"):
        kv.evict(0, d_w, d_n, 8, 1, 4, d_w, None)
    synchronize()
    for a, b in zip(kv.read(0, 0, 32), rows[0, 0]):
        np.testing.assert_array_equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("keep", [12288, 12289])
def test_long_lists(hd, keep):
    """Around the longest list of kept slots that one launch holds, more slots than a block has in registers."""
    rng = np.random.default_rng(keep)
    cap = 20001
    kv, rows = filled(rng, 1, cap, 1, hd)
    w = weights(rng, 1, 1, cap)
    for kept in (True, False):
        check(kv, rows, w, [cap], keep, 7, 1000, run(kv, w, [cap], keep, 7, 1000, kept=kept))
        kv, rows = filled(rng, 1, cap, 1, hd)
