"""Two layers of a model over the paged cache, as a server runs them: int8 CQ projections (multi-matrix plans), heads normed,
rotated and stored, attention of the ragged batch, the output projection; each stage against the oracle or the formula on
the stage's own GPU input (tolerances: tests/test_heads_gpu.py, tests/test_paged_gpu.py), eager and replayed from one graph.
"""
import numpy as np
import pytest

import oracle
from openneedle_amd.cq import CQMatrix, Plan
from openneedle_amd.device import DeviceArray, Graph, Stream, synchronize
from openneedle_amd.heads import rotary_frequencies
from openneedle_amd.paged import PagedCache
from tests.cases import baseline
from tests.test_heads_gpu import heads_of
from tests.test_paged import Pool
from tests.test_paged_gpu import Batch, Rows, ints, upload

pytestmark = pytest.mark.gpu

LAYERS, HEADS, KVHEADS, HD, HIDDEN, PAGE = 2, 8, 4, 64, 512, 16


class Model:
    def __init__(self, rng, requests, tokens, pages, width):
        self.requests, self.tokens, self.width = requests, tokens, width
        self.stream = Stream()
        self.kv = PagedCache(LAYERS, pages, PAGE, KVHEADS, HD)
        self.pool = Pool(pages, PAGE, requests, width)
        self.rows = [Rows(self.kv, i) for i in range(LAYERS)]
        self.freq = rotary_frequencies(10000.0, HD)
        self.gains = rng.normal(size=(LAYERS, 2, HD)).astype(np.float32) * 0.2
        self.step_d = dict(counts=ints(np.zeros(requests)), lengths=ints(np.zeros(requests)),
                           tables=ints(np.full((requests, width), -1)), starts=ints(np.zeros(requests + 1)),
                           firsts=ints(np.zeros(requests)), slots=ints(np.zeros(tokens)), positions=ints(np.zeros(tokens)))
        self.d_freq = upload(self.freq, np.float64)
        self.layers, x = [], upload(np.zeros((tokens, HIDDEN)))
        for i in range(LAYERS):
            host, mats = {}, {}
            for j, (name, n) in enumerate((("q", HEADS * HD), ("k", KVHEADS * HD), ("v", KVHEADS * HD), ("o", HIDDEN))):
                packed, norms, cb, _ = baseline(4, n, HIDDEN, seed=100 * i + j)
                host[name], mats[name] = (packed, norms, cb), CQMatrix(packed, norms, (n, HIDDEN), 4, 32, cb)
            d = {n: upload(np.zeros((tokens, w))) for n, w in (("q", HEADS * HD), ("k", KVHEADS * HD), ("v", KVHEADS * HD),
                                                               ("turned", HEADS * HD), ("keys", KVHEADS * HD), ("att", HEADS * HD), ("o", HIDDEN))}
            d["x"], d["qg"], d["kg"] = x, upload(self.gains[i, 0]), upload(self.gains[i, 1])
            self.layers.append(dict(host=host, mats=mats, d=d, qkv=Plan([mats[n] for n in "qkv"], [x] * 3, [d[n] for n in "qkv"], tokens, int8=True),
                                    o=Plan([mats["o"]], [d["att"]], [d["o"]], tokens, int8=True)))
            x = d["o"]

    def issue(self, count):
        s = self.step_d
        self.kv.extend(self.requests, s["counts"], self.tokens, s["lengths"], s["tables"], self.width, s["starts"], s["firsts"],
                       s["slots"], s["positions"], stream=self.stream)
        for i, layer in enumerate(self.layers):
            d = layer["d"]
            layer["qkv"].run(self.stream)
            self.kv.store_rotated(i, d["q"], d["k"], d["v"], HEADS, self.tokens, s["positions"], s["slots"], self.d_freq, HD,
                                  d["qg"], d["kg"], d_q_out=d["turned"], d_k_out=d["keys"], stream=self.stream)
            self.kv.attention(i, d["turned"], d["att"], HEADS, self.requests, self.tokens, count, s["starts"], s["firsts"],
                              s["tables"], self.width, stream=self.stream)
            layer["o"].run(self.stream)

    def feed(self, rng, counts):
        self.x = rng.normal(size=(self.tokens, HIDDEN)).astype(np.float32)
        self.layers[0]["d"]["x"].upload(self.x)
        self.step_d["counts"].upload(np.asarray(counts, np.int32))
        synchronize()

    def verify(self, counts, count):
        synchronize()
        starts, firsts, slots, positions = self.pool.extend(counts, self.tokens)
        np.testing.assert_array_equal(self.step_d["slots"].to_host(np.int32, self.tokens), slots)
        live = np.array(positions) >= 0
        for i, layer in enumerate(self.layers):
            got = {n: layer["d"][n].to_host(np.float32, (self.tokens, w)) for n, w in
                   (("x", HIDDEN), ("q", HEADS * HD), ("k", KVHEADS * HD), ("v", KVHEADS * HD), ("turned", HEADS * HD),
                    ("keys", KVHEADS * HD), ("att", HEADS * HD), ("o", HIDDEN))}
            for name, src in (("q", "x"), ("k", "x"), ("v", "x"), ("o", "att")):
                packed, norms, cb = layer["host"][name]
                np.testing.assert_array_equal(got[name], oracle.sdot_linear(packed, norms, (packed.shape[0], HIDDEN), 4, 32, cb,
                                                                            got[src], 8), err_msg=f"layer {i}: {name}")
            by_head = {n: got[n].reshape(self.tokens, -1, HD) for n in ("q", "k", "v", "turned", "keys", "att")}
            for src, to, gain in (("q", "turned", self.gains[i, 0]), ("k", "keys", self.gains[i, 1])):
                want, tol = heads_of(by_head[src][live], np.array(positions)[live], gain, self.freq, 1e-6)
                assert (np.abs(by_head[to][live] - want) <= tol).all()
            self.rows[i].put([s if ok else -1 for s, ok in zip(slots, live)], by_head["keys"], by_head["v"])
            self.rows[i].same()
            b = Batch.__new__(Batch)
            b.kv, b.rows, b.group, b.tables, b.starts, b.q = self.kv, self.rows[i], HEADS // KVHEADS, np.array(self.pool.tables), starts, by_head["turned"]
            b.counts, b.past = [c if f >= 0 else 0 for c, f in zip(counts, firsts)], firsts
            b.check(by_head["att"], many=count > 32)


def test_two_layers_eager_and_replayed():
    rng = np.random.default_rng(31)
    m = Model(rng, 4, 72, 60, 12)
    graph = None
    steps = [[70, 0, 1, 0], [1, 40, 3, 2], [1, 1, 1, 1], [1, 1, 66, 1], [1, 1, 1, 1]]
    for i, counts in enumerate(steps):
        m.feed(rng, counts)
        if i == 1:  # the step has run once: from here on it is replayed
            with Graph.capture(m.stream) as graph:
                m.issue(72)
        if graph is None:
            m.issue(72)
        else:
            graph.launch(m.stream)
        m.verify(counts, 72)
        if i == 2:  # a request ends, its pages go to the others
            keep = [0, -1, -1, -1]
            m.kv.trim(4, ints(keep), m.step_d["lengths"], m.step_d["tables"], m.width, stream=m.stream)
            m.pool.trim(keep)
    graph.close()
