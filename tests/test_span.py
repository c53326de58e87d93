"""Host arithmetic of the span attention: which slots a query attends, and the argument rules (no GPU).

The headers hold no HIP types, so they are compiled here with the host compiler and called through ctypes.
"""
import ctypes as ct
import subprocess
from pathlib import Path

import numpy as np
import pytest

from openneedle_amd import _ffi

CSRC = Path(__file__).resolve().parents[1] / "openneedle_amd" / "csrc"

SOURCE = r"""
#include "span_check.h"
#include "span_geom.h"
extern "C" {
int slot(int p, int sinks, int capacity) { return nd::ring_slot(p, sinks, capacity); }
void runs(int first, int last, int sinks, int window, int capacity, int *out) {
    nd::KeyRuns r = nd::ring_runs(first, last, sinks, window, capacity);
    int v[6] = {r.n0, r.begin1, r.n1, r.pinned, r.shift0, r.shift1};
    for (int i = 0; i < 6; ++i) out[i] = v[i];
}
int tiles(int n) { return nd::span_tiles(n); }
const char *window_rule(int c, int s, int k, int h, int n, int sinks, int window) {
    return nd::check_window(c, s, k, h, n, sinks, window);
}
const char *length_rule(int c, int s, int k, int h, int length) { return nd::check_length(c, s, k, h, length); }
const char *prefix_rule(int k, int d, int pc, int pk, int pd, int ps, int seq, int length) {
    return nd::check_prefix(k, d, pc, pk, pd, ps, seq, length);
}
const char *evict_rule(int c, int s, int k, int keep, int sinks, int recent) {
    return nd::check_evict(c, s, k, keep, sinks, recent);
}
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("span")
    (d / "span.cpp").write_text(SOURCE)
    out = d / "span.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=undefined",
                    "-shared", "-fPIC", "-I", str(CSRC), str(d / "span.cpp"), "-o", str(out)], check=True)
    lib = ct.CDLL(str(out))
    for f in (lib.window_rule, lib.length_rule, lib.prefix_rule, lib.evict_rule):
        f.restype = ct.c_char_p
    return lib


def positions_of(host, first, last, sinks, window, capacity):
    """{slot: position} of the two runs, and their slots in order."""
    v = (ct.c_int * 6)()
    host.runs(first, last, sinks, window, capacity, v)
    n0, begin1, n1, pinned, shift0, shift1 = v
    slots = [(j, j if j < pinned else j + shift0) for j in range(n0)] + [(j, j + shift1) for j in range(begin1, begin1 + n1)]
    assert len({s for s, _ in slots}) == len(slots)
    return dict(slots), v


@pytest.mark.parametrize("sinks,window,extra", [(0, 1, 0), (0, 7, 0), (1, 1, 0), (4, 16, 0), (4, 16, 5), (9, 3, 1), (64, 65, 0),
                                                (3, 130, 40)])
@pytest.mark.parametrize("count", [1, 2, 5, 33])
def test_runs_hold_the_attended_positions_once(host, sinks, window, extra, count):
    capacity = sinks + window + count - 1 + extra
    starts = list(range(-count - 1, 3 * capacity + 3)) + [2 ** 31 - 1 - count, 2 ** 31 - 2 - capacity]
    for first in starts:
        last = first + count - 1
        got, _ = positions_of(host, first, last, sinks, window, capacity)
        low = max(first, 0) - window + 1
        want = set(range(min(sinks, last + 1))) | set(range(max(sinks, low), last + 1)) if last >= 0 else set()
        assert set(got.values()) == want, first
        for slot, p in got.items():
            assert 0 <= slot < capacity
            assert slot == (p if p < sinks else sinks + (p - sinks) % (capacity - sinks)) == host.slot(p, sinks, capacity)


@pytest.mark.parametrize("sinks,window", [(0, 1), (4, 60), (4, 61), (65, 64), (1, 256), (17, 999)])
@pytest.mark.parametrize("count", [1, 6])
def test_tiles_stay_below_the_planned_number(host, sinks, window, count):
    """The pieces are planned for span_tiles(sinks + window + count - 1) + 1 tiles."""
    capacity = sinks + window + count - 1
    most = host.tiles(capacity) + 1
    for first in range(-2, 3 * capacity):
        _, v = positions_of(host, first, first + count - 1, sinks, window, capacity)
        assert host.tiles(v[0]) + host.tiles(v[2]) <= most


def test_the_newest_position_ends_its_run(host):
    """The store inside a one-token launch goes by this: run 1's end, or run 0's where that holds ring slots or run 1 is
    empty."""
    for sinks, window, extra in [(0, 1, 0), (0, 5, 2), (4, 16, 0), (4, 16, 9), (70, 3, 0)]:
        capacity = sinks + window + extra
        for p in range(3 * capacity + 2):
            _, (n0, begin1, n1, pinned, _, _) = positions_of(host, p, p, sinks, window, capacity)
            in1 = n1 > 0 and not n0 > pinned
            assert (begin1 + n1 - 1 if in1 else n0 - 1) == host.slot(p, sinks, capacity)


def test_argument_rules(host):
    assert host.window_rule(20, 2, 2, 4, 1, 4, 16) is None
    assert host.window_rule(20, 2, 2, 4, 0, 4, 16) is None
    assert host.window_rule(24, 2, 2, 32, 5, 4, 16) is None
    for args, word in [((20, 2, 2, 3, 1, 4, 16), b"multiple"), ((20, 2, 2, 0, 1, 4, 16), b"multiple"),
                       ((20, 2, 2, 34, 1, 4, 16), b"16 query heads"), ((20, 2, 2, 4, -1, 4, 16), b"count"),
                       ((20, 2, 2, 4, 1, -1, 16), b"sinks"), ((20, 2, 2, 4, 1, 4, 0), b"window"),
                       ((20, 2, 2, 4, 2, 4, 16), b"capacity"), ((20, 2, 2, 4, 1, 2 ** 31 - 1, 2 ** 31 - 1), b"capacity"),
                       ((2 ** 30, 64, 2, 32, 2 ** 20, 4, 16), b"rows"), ((20, 70000, 1, 1, 1, 4, 16), b"65535"),
                       ((2 ** 25, 64, 2, 32, 2 ** 14 + 1, 4, 16), b"2^25"), ((20, 2 ** 15, 2 ** 4, 2 ** 8, 1, 4, 16), b"2^22")]:
        assert word in host.window_rule(*args), args
    assert host.length_rule(20, 2, 2, 4, 0) is None and host.length_rule(20, 2, 2, 4, 20) is None
    assert b"length" in host.length_rule(20, 2, 2, 4, 21) and b"length" in host.length_rule(20, 2, 2, 4, -1)
    assert host.prefix_rule(2, 64, 100, 2, 64, 3, 2, 100) is None
    for args, word in [((2, 64, 100, 4, 64, 3, 2, 100), b"geometry"), ((2, 64, 100, 2, 32, 3, 2, 100), b"geometry"),
                       ((2, 64, 100, 2, 64, 3, 3, 100), b"sequence"), ((2, 64, 100, 2, 64, 3, -1, 100), b"sequence"),
                       ((2, 64, 100, 2, 64, 3, 2, 101), b"prefix length"), ((2, 64, 100, 2, 64, 3, 2, -1), b"prefix length")]:
        assert word in host.prefix_rule(*args), args
    assert host.evict_rule(20, 2, 2, 20, 4, 16) is None
    for args, word in [((20, 2, 2, 21, 4, 16), b"capacity"), ((20, 2, 2, 0, 0, 0), b"keep"), ((20, 2, 2, 8, -1, 2), b">= 0"),
                       ((20, 2, 2, 8, 1, -2), b">= 0"), ((20, 2, 2, 8, 4, 5), b"exceeds keep"),
                       ((20, 2, 2, 8, 2 ** 31 - 1, 2 ** 31 - 1), b"exceeds keep"), ((20, 2, 70000, 8, 4, 4), b"65535")]:
        assert word in host.evict_rule(*args), args


def test_null_handles_are_refused():
    lib = _ffi.lib()
    assert lib.needle2_gpu_attention_window(None, 0, None, None, 4, 1, None, 4, 16, None, None, None) == -1
    assert "null KV cache" in _ffi.last_error()
    assert lib.needle2_gpu_attention_shared(None, 0, None, 0, 1, None, None, 4, 1, None, None, None, None) == -1
    assert lib.needle2_gpu_attention_weights(None, 0, None, None, None, 4, 1, None, None, None, None) == -1
    assert lib.needle2_gpu_kv_evict(None, 0, None, None, 1, 0, 0, None, None, None, None) == -1
    assert lib.needle2_gpu_kv_layer(None, 0, None, None, None, None) == -1
    assert "null KV cache" in _ffi.last_error()


def test_kept_order_matches_a_plain_sort():
    """The oracle of the eviction tests itself: stable, lowest slots first among equals, NaN last."""
    from tests.test_evict_gpu import kept_slots
    w = np.array([0, 5, 1, np.nan, 1, -0.0, 0.0, 1, -2, 9], np.float32)
    assert kept_slots(w, 10, 6, 1, 1) == [0, 1, 2, 4, 7, 9]
    assert kept_slots(w, 10, 7, 1, 1) == [0, 1, 2, 4, 5, 7, 9]
    assert kept_slots(w, 10, 9, 1, 1) == [0, 1, 2, 4, 5, 6, 7, 8, 9]
    assert kept_slots(w, 5, 6, 1, 1) == [0, 1, 2, 3, 4]
