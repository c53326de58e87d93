"""Eviction of all layers of a cache whose sequences share one array of lengths."""
import numpy as np
import pytest

from openneedle_amd.device import DeviceArray, synchronize
from tests.test_evict_gpu import check, filled, weights


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [True, False])
def test_every_layer_is_cut_from_the_lengths_before(in_place):
    """A record per layer, in place or not; the lengths go to an array of their own, the last layer's call may write them
    over the old ones."""
    rng = np.random.default_rng(3)
    layers, seqs, kvh, cap, hd, keep, sinks, recent = 3, 4, 2, 500, 64, 120, 4, 30
    kv, rows = filled(rng, seqs, cap, kvh, hd, layers)
    w = [weights(rng, seqs, kvh, cap) for _ in range(layers)]
    lengths = np.array([500, 120, 121, 77], np.int32)
    d_w = [DeviceArray.from_host(a) for a in w]
    d_cut = d_w if in_place else [DeviceArray.from_host(np.full(a.shape, 7, np.float32)) for a in w]
    d_n, d_m = DeviceArray.from_host(lengths), DeviceArray.from_host(np.full(seqs, 7, np.int32))
    for layer in range(layers):
        last = layer == layers - 1
        kv.evict(layer, d_w[layer], d_n, keep, sinks, recent, d_cut[layer], d_n if last else d_m)
    synchronize()
    np.testing.assert_array_equal(d_n.to_host(np.int32, seqs), d_m.to_host(np.int32, seqs))
    for layer in range(layers):
        got = (d_cut[layer].to_host(np.float32, w[layer].shape), d_n.to_host(np.int32, seqs), None)
        check(kv, rows, w[layer], lengths, keep, sinks, recent, got, layer=layer)
