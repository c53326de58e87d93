"""How the span attention's launches are cut, and that the GPU tests of the many-row kernel reach it (no GPU).

The plan is arithmetic on plain integers: it is compiled here with the host compiler, for a device of 256 compute units.
"""
import ctypes as ct
import subprocess
from pathlib import Path

import pytest

from tests import test_span_wide_gpu as wide

CSRC = Path(__file__).resolve().parents[1] / "openneedle_amd" / "csrc"

SOURCE = r"""
#include "span_plan.h"
static void put(const nd::SpanCut &c, int *out) {
    const int v[5] = {c.wide, c.splits, c.per, c.waves, c.groups};
    for (int i = 0; i < 5; ++i) out[i] = v[i];
}
extern "C" {
void window_cut(int hd, int capacity, int seqs, int kvheads, int heads, int count, int sinks, int window, int *out) {
    put(nd::cut_window(256, hd, capacity, seqs, kvheads, heads, count, sinks, window), out);
}
void prefix_cut(int hd, int seqs, int kvheads, int heads, int length, int *out) {
    put(nd::cut_prefix(256, hd, seqs, kvheads, heads, length), out);
}
void own_cut(int hd, int seqs, int kvheads, int heads, int length, int *out) {
    put(nd::cut_own(256, hd, seqs, kvheads, heads, length, true), out);
}
int tiles(int n) { return nd::span_tiles(n); }
int wide_tiles(int n) { return nd::wide_tiles(n); }
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(SOURCE)
    out = d / "plan.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", str(CSRC), str(d / "plan.cpp"),
                    "-o", str(out)], check=True)
    return ct.CDLL(str(out))


def call(f, *args):
    v = (ct.c_int * 5)()
    f(*args, v)
    return dict(zip(("wide", "splits", "per", "waves", "groups"), v))


def window(host, hd, shape, extra=0):
    seqs, kvh, group, count, sinks, span = shape
    return call(host.window_cut, hd, sinks + span + count - 1 + extra, seqs, kvh, kvh * group, count, sinks, span)


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_the_many_row_kernels_tests_reach_it(host, hd):
    for shape in wide.EDGES:
        for extra in (0, shape[5] % 3, 90):
            assert window(host, hd, shape, extra)["wide"], shape
    assert window(host, hd, wide.LONG, 7)["wide"] and window(host, hd, wide.LONG)["splits"] > 8
    one = window(host, hd, wide.PIECE)
    assert one["wide"] and one["splits"] == 1
    for n, kvh, group, length in [*wide.PREFIXES, wide.GRAPH_PREFIX]:
        assert call(host.prefix_cut, hd, n, kvh, kvh * group, length)["wide"], (n, kvh, group, length)
    n, kvh, group, length = wide.PREFIXES[2]
    assert call(host.prefix_cut, hd, n, kvh, kvh * group, length)["per"] > 1
    one, more = ((window(host, 64, s)["splits"] * s[1] * s[2] * s[3]) for s in (wide.GRAPH_WINDOW, wide.GRAPH_OUTGROWN))
    assert more > one  # records


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_pieces_cover_the_tiles(host, hd):
    """Every tile is in a piece, and no more pieces than the join takes (1024 with a prefix and own slots together)."""
    for seqs in (1, 2, 7, 64, 1000):
        for kvh, group in ((1, 1), (4, 2), (8, 4), (2, 16)):
            for n in (0, 1, 63, 64, 65, 1000, 8192, 65537, 1 << 20):
                far, own = (call(f, hd, seqs, kvh, kvh * group, n) for f in (host.prefix_cut, host.own_cut))
                for c in (far, own):
                    assert c["splits"] >= 1 and c["splits"] * c["per"] >= (host.wide_tiles if c["wide"] else host.tiles)(n)
                    assert c["splits"] <= 512 and c["waves"] in (4, 8) and (c["groups"] in range(1, 5)) == bool(c["wide"])
                assert not own["wide"]
                for count in (1, 5, 40, 999):
                    c = window(host, hd, (seqs, kvh, group, count, 4, max(n, 1)))
                    tokens = -(-(128 if c["wide"] else 16) // group) + 1  # of a block, whose keys are two runs
                    keys = 4 + max(n, 1) + min(count, tokens) - 1
                    assert c["splits"] * c["per"] >= (host.wide_tiles if c["wide"] else host.tiles)(keys) + 1
                    assert not c["wide"] or (c["groups"] == 4 and count * group > 16)
