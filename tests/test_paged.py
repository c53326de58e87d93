"""Host arithmetic of the paged cache: which positions a row tile attends, how the attention is cut, the argument rules,
refusals that need no GPU, and the tests' own model of the tables (no GPU).

The headers hold no HIP types, so they are compiled here with the host compiler and called through ctypes.
"""
import ctypes as ct
import subprocess
from pathlib import Path

import numpy as np
import pytest

from openneedle_amd import _ffi
from openneedle_amd.heads import rotary_frequencies

CSRC = Path(__file__).resolve().parents[1] / "openneedle_amd" / "csrc"

SOURCE = r"""
#include "paged_check.h"
#include "paged_plan.h"
extern "C" {
void runs(int first, int last, int window, int tile, int *out) {
    nd::KeyRuns r = nd::page_runs(first, last, window, tile);
    int v[6] = {r.n0, r.begin1, r.n1, r.pinned, r.shift0, r.shift1};
    for (int i = 0; i < 6; ++i) out[i] = v[i];
}
void cut(int hd, int requests, int tokens, int count, int kvheads, int group, int length, int window, int *out) {
    nd::PagedCut c = nd::cut_paged(256, hd, requests, tokens, count, kvheads, group, length, window);
    int v[10] = {c.small, c.row_tiles, c.rows.splits, c.rows.per, c.rows.waves, c.wide_blocks, c.wide.splits, c.wide.per, c.round,
                 int(c.few_records * c.rows.splits + c.wide_records * c.wide.splits)};
    for (int i = 0; i < 10; ++i) out[i] = v[i];
}
const char *pages_rule(int l, int n, int p, int k, int d) { return nd::check_pages(l, n, p, k, d); }
const char *requests_rule(int r, int w, int p) { return nd::check_requests(r, w, p); }
const char *tokens_rule(int t) { return nd::check_tokens(t); }
const char *rows_rule(size_t at, int stride, int h, int d) { return nd::check_rows((const void *)at, stride, h, d); }
const char *turn_rule(int h, int k, int d, int t, float eps, int rotary) { return nd::check_turn(h, k, d, t, eps, rotary); }
const char *attention_rule(int k, int h, int r, int t, int c, int l, int w) {
    return nd::check_paged_attention(k, h, r, t, c, l, w);
}
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    (d / "paged.cpp").write_text(SOURCE)
    out = d / "paged.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=undefined",
                    "-shared", "-fPIC", "-I", str(CSRC), str(d / "paged.cpp"), "-o", str(out)], check=True)
    lib = ct.CDLL(str(out))
    for f in (lib.pages_rule, lib.requests_rule, lib.tokens_rule, lib.rows_rule, lib.turn_rule, lib.attention_rule):
        f.restype = ct.c_char_p
    lib.rows_rule.argtypes = [ct.c_size_t, ct.c_int, ct.c_int, ct.c_int]
    lib.turn_rule.argtypes = [ct.c_int] * 4 + [ct.c_float, ct.c_int]
    return lib


@pytest.mark.parametrize("tile", [32, 64])
@pytest.mark.parametrize("window", [0, 1, 5, 64, 1000])
def test_runs_hold_every_attended_position(host, tile, window):
    """One run, from a multiple of a tile at most a tile before the first row's window, to the last row's own position."""
    for count in (1, 2, 33, 100):
        for first in [*range(0, 3 * tile), 999, 1000, 1001, 2 ** 30 - count]:
            v = (ct.c_int * 6)()
            host.runs(first, first + count - 1, window, tile, v)
            n0, begin, n, pinned, s0, s1 = v
            low = max(0, first - window + 1) if window else 0
            assert n0 == pinned == s0 == s1 == 0 and begin % tile == 0 and begin + n == first + count
            assert begin <= low < begin + tile
    host.runs(-1, 4, window, tile, v)
    assert not any(v)


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_the_cut_holds_every_row(host, hd):
    """Blocks for every row, no more pieces than the join takes, no more blocks than a grid."""
    for requests, counts in [(1, [1]), (1, [2000]), (64, [1] * 64), (8192, [1] * 8192), (8192, [90] + [1] * 8191), (8192, [300] + [1] * 8191), (7, [5] * 7), (51, [1] * 48 + [700, 3, 999]),
                             (3, [0, 40, 0]), (2, [1, 100000]), (2, [1, 8000]), (3, [1, 60, 3000])]:
        for kvheads, group in ((1, 1), (4, 2), (8, 4), (2, 16), (1, 13), (512, 1)):
            tokens, most = sum(counts), max(counts)
            if tokens * kvheads * group > 1 << 25:
                continue
            for length, window in ((max(1, most), 0), (8192 + most, 0), (1 << 20, 0), (1 << 20, 500)):
                v = (ct.c_int * 10)()
                host.cut(hd, requests, tokens, most, kvheads, group, length, window, v)
                small, row_tiles, splits, per, waves, wide_blocks, wide_splits, wide_per, round, records = v
                assert splits >= 1 and per >= 1 and waves in (4, 8) and splits <= 1024
                assert min(most * group, small) <= row_tiles * 16
                assert round == 0 or requests <= 512
                assert 0 <= records <= 1 << 18  # of the scratch: 140 MB at most
                assert (row_tiles * requests * splits + wide_blocks * wide_splits) * kvheads < 1 << 24
                if most * group > small:
                    need, start = 0, 0
                    for r, c in enumerate(counts):
                        if requests > 512:  # found without their lengths
                            need = max(need, start * group // 128 + r + -(-c * group // 128))
                            start += c
                        elif c * group > small:
                            need += -(-c * group // 128)
                    assert wide_blocks >= need and 1 <= wide_splits <= 1024 and wide_per >= 1 and waves == 4


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_the_tests_of_many_rows_reach_their_kernel(host, hd):
    from tests.test_paged_wide_gpu import SHAPES, grown
    for kvheads, group, counts, past in [*SHAPES, (1, 2, [90, 1, 130], [0]), (1, 2, [70, 1, 2, 40], [6000]), (1, 2, [80, 70, 66], [200]),
                                         (1, 2, [70, 1], [150])]:
        counts = grown(hd, group, counts)
        v = (ct.c_int * 10)()
        host.cut(hd, len(counts), sum(counts), max(counts), kvheads, group, max(past) + max(counts), 0, v)
        small, row_tiles, _, _, _, wide_blocks, *_ = v
        assert wide_blocks and max(counts) * group > small, (kvheads, group, counts)
        assert len(counts) == 1 or row_tiles * 16 >= small


def test_the_tests_of_ordered_requests_reach_the_order(host):
    from tests.test_paged_gpu import ORDERED
    for requests, kvheads in ORDERED:
        for count in (1, 2):
            v = (ct.c_int * 10)()
            host.cut(32, requests, requests * count, count, kvheads, 2, 1152, 0, v)
            assert v[8] > 0, (requests, kvheads)
    host.cut(64, 1, 1, 1, 1, 2, 1 << 20, 0, v)
    assert v[8] == 0


def test_the_test_of_many_pieces_has_them(host):
    from tests.test_paged_gpu import MANY_PIECES
    for hd, past in MANY_PIECES:
        v = (ct.c_int * 10)()
        host.cut(hd, 1, 1, 1, 1, 2, past + 1, 0, v)
        assert v[2] >= 64, (hd, past, v[2])


def test_the_graphs_with_records_have_them(host):
    """Each captured step has records of both kinds that it can have, every later call more than fit the scratch before it,
    and the requests of the test have keys for several pieces."""
    from tests.test_paged_gpu import OUTGROWN, RECORDED as c, RECORDED_COUNTS
    calls = [(c["tokens"], n) for n in RECORDED_COUNTS] + [(OUTGROWN["tokens"], OUTGROWN["count"])]
    for counts in ((1, 1), (130, 1)):  # and those of a first call that is captured
        v = (ct.c_int * 10)()
        host.cut(64, 2, sum(counts), max(counts), 2, 2, 3001, 0, v)
        assert v[9] > 0 and v[2] > 1 and v[3] * 64 < 900 and (max(counts) == 1 or (v[6] > 1 and v[7] * 32 < 1200))
    held_records = held_rows = 0
    for tokens, count in calls:
        v = (ct.c_int * 10)()
        host.cut(c["hd"], c["requests"], tokens, count, c["kvheads"], c["group"], c["width"] * c["page"], 0, v)
        small, row_tiles, splits, per, _, wide_blocks, wide_splits, wide_per, _, records = v
        rows = c["requests"] * c["kvheads"] * row_tiles * 16
        assert splits > 1 and per * 64 < 390  # (keys of the second longest request)
        if count > 1:
            rows += tokens * c["kvheads"] * c["group"]
            assert wide_blocks and wide_splits > 1 and wide_per * 32 < 390 and count * c["group"] > small
        assert records > held_records and rows > held_rows, (tokens, count)
        # (the scratch at least doubles)
        held_records, held_rows = max(records, 2 * held_records), max(rows, 2 * held_rows)


def test_argument_rules(host):
    assert host.pages_rule(1, 10, 16, 2, 64) is None and host.pages_rule(1, 2 ** 27 - 1, 16, 1, 32) is None
    for args, word in [((0, 10, 16, 2, 64), b"positive"), ((1, 0, 16, 2, 64), b"positive"), ((1, 10, 16, 0, 64), b"positive"),
                       ((1, 10, 8, 2, 64), b"page_size"), ((1, 10, 24, 2, 64), b"page_size"), ((1, 10, 512, 2, 64), b"page_size"),
                       ((1, 10, 16, 2, 96), b"head_dim"), ((1, 10, 16, 70000, 64), b"65535"), ((1, 10, 256, 40000, 128), b"2^31 bytes"), ((1, 2 ** 27, 16, 2, 64), b"2^31")]:
        assert word in host.pages_rule(*args), args
    # 2^22 layers of 2^20 pages of over 2^22 bytes: past 2^64, where the sizes wrap
    assert b"2^46" in host.pages_rule(1 << 22, 1 << 20, 256, 1 << 6, 128)
    assert b"2^46" in host.pages_rule(2 ** 31 - 1, 2 ** 27 - 1, 16, 65535, 128)
    assert host.pages_rule(64, 1 << 20, 16, 8, 128) is None
    assert host.requests_rule(0, 1, 16) is None and host.requests_rule(8192, 2 ** 26, 16) is None
    for args, word in [((-1, 1, 16), b"8192"), ((8193, 1, 16), b"8192"), ((1, 0, 16), b"width"), ((1, 2 ** 26 + 1, 16), b"2^30")]:
        assert word in host.requests_rule(*args), args
    assert host.tokens_rule(0) is None and host.tokens_rule(2 ** 25) is None
    assert b"2^25" in host.tokens_rule(-1) and b"2^25" in host.tokens_rule(2 ** 25 + 1)
    assert host.rows_rule(1 << 40, 256, 4, 64) is None and host.rows_rule(1 << 40, 260, 4, 64) is None
    for args, word in [((1 << 40, 252, 4, 64), b"stride"), ((1 << 40, 258, 4, 64), b"16 bytes"), ((8, 256, 4, 64), b"16 bytes"),
                       ((1 << 40, 0, 4, 64), b"stride")]:
        assert word in host.rows_rule(*args), args
    assert host.turn_rule(8, 4, 64, 10, 1e-6, 64) is None and host.turn_rule(0, 0, 32, 0, 0.0, 0) is None
    for args, word in [((8, 4, 48, 10, 1e-6, 32), b"head_dim"), ((-1, 4, 64, 10, 1e-6, 64), b"65535"),
                       ((8, 70000, 64, 10, 1e-6, 64), b"65535"), ((8, 4, 64, -1, 1e-6, 64), b"2^25"), ((8, 4, 64, 1, -1.0, 64), b"eps"),
                       ((8, 4, 64, 1, float("nan"), 64), b"eps"), ((8, 4, 64, 1, 1e-6, 66), b"rotary"),
                       ((8, 4, 64, 1, 1e-6, 7), b"rotary"), ((8, 4, 64, 1, 1e-6, -2), b"rotary")]:
        assert word in host.turn_rule(*args), args
    assert host.attention_rule(2, 8, 3, 10, 10, 0, 0) is None and host.attention_rule(2, 32, 3, 10, 0, 7, 9) is None
    for args, word in [((2, 3, 3, 10, 1, 0, 0), b"multiple"), ((2, 0, 3, 10, 1, 0, 0), b"multiple"), ((2, 34, 3, 10, 1, 0, 0), b"16 query"),
                       ((2, 4, 3, 10, 11, 0, 0), b"count"), ((2, 4, 3, 10, -1, 0, 0), b"count"), ((2, 4, 3, 10, 1, -1, 0), b"length"),
                       ((2, 4, 3, 10, 1, 0, -1), b"window"), ((256, 4096, 8192, 10, 1, 0, 0), b"2^22"),
                       ((2, 32, 3, 2 ** 21, 1, 0, 0), b"2^25")]:
        assert word in host.attention_rule(*args), args


def test_calls_without_a_cache_are_refused():
    lib = _ffi.lib()
    p = ct.c_int()
    assert lib.needle2_gpu_pages_extend(None, 0, None, 0, None, None, 1, None, None, None, None, None) == -1
    assert "null paged cache" in _ffi.last_error()
    assert lib.needle2_gpu_pages_trim(None, 0, None, None, None, 1, None) == -1
    assert lib.needle2_gpu_pages_store(None, 0, None, 64, None, 64, 0, None, None) == -1
    assert lib.needle2_gpu_pages_attention(None, 0, None, None, 2, 0, 0, 0, None, None, None, 1, 0, 0, None) == -1
    assert lib.needle2_gpu_pages_free(None, ct.byref(p), None) == -1 and lib.needle2_gpu_pages_reset(None, None) == -1
    assert lib.needle2_gpu_pages_layer(None, 0, None) == -1 and lib.needle2_gpu_pages_storage_bytes(None) == 0
    assert "null paged cache" in _ffi.last_error()
    assert lib.needle2_gpu_pages_create(1, 10, 20, 1, 64) is None and "page_size" in _ffi.last_error()


def test_heads_refuses_before_any_launch():
    """(No device is touched: every call here is refused, or has no tokens or no rows.)"""
    lib, at = _ffi.lib(), 1 << 40

    def heads(q=at, qs=256, qo=at, qos=256, h=4, k=at, ks=128, ko=at, kos=128, kvh=2, hd=64, n=3, pos=at, qg=None, kg=None, eps=0.0,
              freq=at, rotary=64):
        return lib.needle2_gpu_heads(q, qs, qo, qos, h, k, ks, ko, kos, kvh, hd, n, pos, qg, kg, eps, freq, rotary, None)

    for args, word in [(dict(q=None), "null q"), (dict(qo=None), "null q"), (dict(k=None), "null k"), (dict(ko=None), "output of k"),
                       (dict(pos=None), "positions"), (dict(freq=None), "positions"), (dict(qs=252), "stride"), (dict(kos=130), "16 bytes"),
                       (dict(k=at + 4), "16 bytes"), (dict(qg=at + 8), "gains"), (dict(rotary=65), "rotary"), (dict(hd=80), "head_dim"),
                       (dict(qo=at, qos=260), "one stride"), (dict(ko=at, kos=132), "one stride")]:
        assert heads(**args) == -1 and word in _ffi.last_error(), args
    assert heads(n=0, q=None, k=None, pos=None, freq=None) == 0
    assert heads(h=0, kvh=0, q=None, qo=None, k=None) == 0


def test_frequencies():
    f = rotary_frequencies(10000.0, 8)
    np.testing.assert_allclose(f, [1, 0.1, 0.01, 0.001], rtol=1e-15)
    assert f.dtype == np.float64 and rotary_frequencies(10000.0, 0).shape == (0,)


class Pool:
    """The paged cache's tables on the host, entry by entry."""

    def __init__(self, pages, page, requests, width):
        self.page, self.width, self.stack = page, width, list(range(pages))[::-1]
        self.lengths, self.tables = [0] * requests, [[-1] * width for _ in range(requests)]

    def extend(self, counts, tokens):
        starts, firsts, slots, positions = [0], [], [-1] * tokens, [-1] * tokens
        left, asked, begin = len(self.stack), 0, 0
        for r, c in enumerate(counts):
            c, n = max(c, 0), self.lengths[r]
            fits = 0 <= n <= n + c <= self.width * self.page
            new = range(-(-n // self.page), -(-(n + c) // self.page)) if fits else range(0)
            asked += len(new)
            ok = fits and begin + c <= tokens and (len(new) == 0 or asked <= left)
            firsts.append(n if ok else -1)
            if ok:
                for i in new:
                    self.tables[r][i] = self.stack.pop()
                for i in range(c):
                    positions[begin + i] = n + i
                    slots[begin + i] = self.tables[r][(n + i) // self.page] * self.page + (n + i) % self.page
                self.lengths[r] = n + c
            begin += c
            starts.append(min(begin, tokens))
        return starts, firsts, slots, positions

    def trim(self, keep):
        gone = []
        for r, k in enumerate(keep):
            k = self.lengths[r] if k < 0 else min(k, self.lengths[r])
            for i in range(-(-k // self.page), -(-self.lengths[r] // self.page)):
                gone.append(self.tables[r][i])
                self.tables[r][i] = -1
            self.lengths[r] = k
        self.stack += gone[::-1]


def test_the_model_of_the_tables():
    p = Pool(5, 4, 3, 3)
    assert p.extend([5, 0, 1], 8) == ([0, 5, 5, 6], [0, 0, 0], [0, 1, 2, 3, 4, 8, -1, -1], [0, 1, 2, 3, 4, 0, -1, -1])
    assert p.tables == [[0, 1, -1], [-1] * 3, [2, -1, -1]] and p.stack == [4, 3]
    before = [list(t) for t in p.tables], list(p.stack)
    p.extend([3, 4, -2], 8)
    p.trim([5, -1, 1])
    assert p.lengths == [5, 4, 1]
    p.trim([9, 0, 2])
    assert ([list(t) for t in p.tables], p.stack) == before
    # the second gets none of two pages wanted where one is left, the third needs none
    p.extend([4, 0, 0], 8)
    assert p.extend([0, 5, 3], 8)[1] == [9, -1, 1] and p.lengths == [9, 0, 4] and len(p.stack) == 1
    assert p.extend([4, 0, 0], 8)[1] == [-1, 0, 4]  # past its table
    p.trim([0, 9, -1])
    assert p.lengths == [0, 0, 4]
    p.trim([0, 0, 0])
    assert p.lengths == [0, 0, 0] and sorted(p.stack) == [0, 1, 2, 3, 4]
