"""Norms and rotation of heads against the formula in 64 bits.

Tolerance, per value, in units of 2^-24 relative to the values that it is made of. The sum of squares rounds at most 8 times
along a value's path (2 levels in a lane, 5 between lanes, the square), half of which reaches the root; with eps added, the
root, the quotient, and the products with it and with 1 + gain (itself rounded) a normed value is off by at most 4 + 5 = 9
units and one more for a gain. Sine and cosine: the angle's rest rounded to 32 bits (at most pi / 4, so 2^-25 off), the last
term of the series 1 unit, what the series leave 2^-29: 2 units of 2^-24. A rotated value has one rounded product and one fma
more: 9 + 1 + 2 + 2 = 14 units of |y_j cos| + |y_j' sin| plus, for the sine and cosine's own errors, 2 units of |y_j| + |y_j'|,
so 16 of |y_j| + |y_j'|. Angles are formed in 64 bits from positions below 2^31: 2^-52 of them, below 2^-21 in all.
"""
import numpy as np
import pytest

from openneedle_amd._ffi import GpuError
from openneedle_amd.device import DeviceArray, Graph, Stream, synchronize
from openneedle_amd.heads import rotary_frequencies, rotate_heads

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24


def heads_of(x, positions, gain, freq, eps):
    """(values, tolerances) of x [tokens][heads][head_dim]."""
    y = x.astype(np.float64)
    if gain is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * (1 + gain.astype(np.float64))
    half = len(freq)
    turn = np.asarray(positions, np.float64)[:, None] * freq if half else np.zeros((len(x), 0))
    out, size = y.copy(), np.abs(y)
    a, b = y[..., :half], y[..., half:2 * half]
    c, s = np.cos(turn)[:, None], np.sin(turn)[:, None]
    out[..., :half], out[..., half:2 * half] = a * c - b * s, b * c + a * s
    size[..., :half] = size[..., half:2 * half] = np.abs(a) + np.abs(b)
    far = np.abs(turn).max(initial=0.0) * 2.0 ** -52
    return out, size * (16 * EPS + far) + 1e-45


def upload(a, dtype=np.float32):
    return DeviceArray.from_host(np.asarray(a, dtype))


def run(q, k, positions, qg, kg, freq, eps=1e-6, stream=None, in_place=False):
    d = [upload(q), upload(k), upload(positions, np.int32), upload(freq, np.float64) if len(freq) else None,
         None if qg is None else upload(qg), None if kg is None else upload(kg)]
    outs = (None, None) if in_place else tuple(DeviceArray.from_host(np.full(x.shape, np.nan, np.float32)) for x in (q, k))
    rotate_heads(d[0], d[1], q.shape[1], k.shape[1], q.shape[2], len(q), d[2], d[3], 2 * len(freq), d[4], d[5], eps,
                 d_q_out=outs[0], d_k_out=outs[1], stream=stream)
    synchronize()
    return tuple((x if o is None else o).to_host(np.float32, y.shape) for x, o, y in zip(d, outs, (q, k)))


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("tokens,heads,kvheads", [(1, 8, 4), (1, 1, 1), (7, 15, 5), (700, 5, 1), (1300, 32, 8)])
@pytest.mark.parametrize("cut", [0, 1, 2, 3])
def test_heads(hd, tokens, heads, kvheads, cut):
    """No rotation, whole rows, half of them, an odd number of pairs."""
    rng = np.random.default_rng(hd + tokens + cut)
    rotary = (0, hd, hd // 2, hd - 10)[cut]
    q, k = (rng.normal(size=(tokens, n, hd)).astype(np.float32) * 3 for n in (heads, kvheads))
    qg, kg = (rng.normal(size=hd).astype(np.float32) * 0.3 for _ in "qk")
    freq = rotary_frequencies(500000.0, rotary)
    positions = rng.integers(0, 1 << 20, tokens)
    for in_place in (False, True):
        got = run(q, k, positions, qg, kg, freq, in_place=in_place)
        for g, x, gain in zip(got, (q, k), (qg, kg)):
            want, tol = heads_of(x, positions, gain, freq, 1e-6)
            assert (np.abs(g - want) <= tol).all()


def test_far_positions():
    """Angles of a billion radians, and of every quarter turn."""
    rng = np.random.default_rng(4)
    positions = np.array([0, 1, 2 ** 31 - 1, 2 ** 30 + 1, 10 ** 9, 123456789, 7])
    q = rng.normal(size=(7, 3, 64)).astype(np.float32)
    freq = np.concatenate([np.arange(8) * np.pi / 4, rng.uniform(0, 1, 24)])
    for g, gain in zip(run(q, q, positions, None, None, freq), (None, None)):
        want, tol = heads_of(q, positions, gain, freq, 1e-6)
        assert (np.abs(g - want) <= tol).all()


@pytest.mark.parametrize("eps", [0.0, 1e-6, 1.0])
def test_sizes_of_rows(eps):
    """Rows from the smallest normal numbers to the largest, zeros, one value among zeros."""
    rng = np.random.default_rng(5)
    q = rng.normal(size=(9, 2, 64)).astype(np.float32)
    q *= np.array([1e-12, 1e-6, 1.0, 1e6, 1e12, 1e18, 1e19, 1e25, 1e37], np.float32)[:, None, None]
    q[2, 1] = 0
    q[3, 1] = 0
    q[3, 1, 5] = 1e30
    gain = rng.normal(size=64).astype(np.float32)
    if eps == 0:  # no norm of a row of zeros
        q[2, 1, 0] = 1
    for g in run(q, q, np.arange(9), gain, gain, np.zeros(0), eps):
        want, tol = heads_of(q, np.arange(9), gain, np.zeros(0), eps)
        assert (np.abs(g - want) <= tol).all()


SIZES = [3.3e38, 4.4e37, 1e37, 1e20, 1e19, 1.0, 1e-12, 1e-15, 1e-18, 3e-20, 3e-22, 1e-23, 1e-30, 1e-37, 1e-41]


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("copies", [1, 400])
@pytest.mark.parametrize("cut", [0, 1, 2])
@pytest.mark.parametrize("eps", [0.0, 1e-44, 1e-38, 1e-33, 1e-6, 1e29])
def test_the_norm_over_the_whole_range(hd, copies, cut, eps):
    """Rows from subnormal values to the largest, whose squares pass the range at either end; rows of one such value among
    zeros, or beside values of another size; eps from a subnormal number to one far above a row. Scaled by a power of two a
    row has the errors of any other; only results below the normal numbers are rounded to 2^-149, once before the gain and
    once after it, and once more when they are rotated."""
    rng = np.random.default_rng(hd + cut)
    x = rng.uniform(0.5, 1.0, (len(SIZES), 4, hd)) * rng.choice([-1, 1], (len(SIZES), 4, hd))
    x[:, 1] = np.sign(x[:, 1])  # values of one size
    x[:, 2] = 0
    x[:, 2, hd // 2 + 3] = 1
    x[:, 3, 1:] *= 2.0 ** -rng.integers(0, 70, hd - 1)
    x = np.tile((x * np.array(SIZES)[:, None, None]).astype(np.float32), (copies, 1, 1))
    gain = rng.normal(size=hd).astype(np.float32)
    freq = rotary_frequencies(1e4, (0, hd, hd - 12)[cut])
    positions = np.arange(len(x)) % 97
    eps = float(np.float32(eps))
    want, tol = heads_of(x, positions, gain, freq, eps)
    tol = tol + 2.0 ** -149 * (3 + 2 * np.abs(1 + gain.astype(np.float64)).max())
    for got in run(x, x, positions, gain, gain, freq, eps):
        assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("eps", [0.0, 1e-42, 1e-6])
def test_the_norm_of_zeros(eps):
    """Zeros where eps is not 0; no number where it is, as the formula has it; the rows beside them as they are."""
    rng = np.random.default_rng(3)
    q = rng.normal(size=(5, 3, 64)).astype(np.float32)
    gain, freq = rng.normal(size=64).astype(np.float32), rotary_frequencies(1e4, 64)
    clean = run(q, q, np.arange(5), gain, gain, freq, eps)
    q[1, 2], q[4, 0] = 0, 0
    for g, c in zip(run(q, q, np.arange(5), gain, gain, freq, eps), clean):
        for row in (g[1, 2], g[4, 0]):
            assert np.isnan(row).all() if eps == 0 else not row.any()
        g[1, 2], g[4, 0] = c[1, 2], c[4, 0]
        np.testing.assert_array_equal(g, c)


def test_rows_of_one_projection_and_tokens_left_out():
    """q and k side by side with v; tokens at negative positions stay as they were; only q, only k; one gain."""
    rng = np.random.default_rng(6)
    n, heads, kvheads, hd = 40, 6, 2, 32
    row = (heads + 2 * kvheads) * hd
    x = rng.normal(size=(n, row)).astype(np.float32)
    positions = rng.integers(0, 999, n)
    positions[[0, 7, 39]] = -1, -2 ** 31, -5
    freq, gain = rotary_frequencies(1e4, hd), rng.normal(size=hd).astype(np.float32)
    for qh, kh in ((heads, kvheads), (heads, 0), (0, kvheads)):
        d, df, dg, dp = upload(x), upload(freq, np.float64), upload(gain), upload(positions, np.int32)
        rotate_heads(d, d.view(heads * hd * 4, 4), qh, kh, hd, n, dp, df, hd, dg, None, q_stride=row, k_stride=row)
        synchronize()
        got, want, tol = d.to_host(np.float32, x.shape), x.astype(np.float64), np.zeros(x.shape)
        live = positions >= 0
        for h, first, g in ((qh, 0, gain), (kh, heads, None)):
            cols = slice(first * hd, (first + h) * hd)
            w, t = heads_of(x[live, cols].reshape(live.sum(), h, hd), positions[live], g, freq, 1e-6)
            want[live, cols], tol[live, cols] = w.reshape(live.sum(), -1), t.reshape(live.sum(), -1)
        assert (np.abs(got - want) <= tol).all()


def test_non_finite_rows_stay_among_themselves():
    rng = np.random.default_rng(7)
    q = rng.normal(size=(3, 4, 64)).astype(np.float32)
    clean = run(q, q, [1, 2, 3], np.ones(64, np.float32), None, rotary_frequencies(1e4, 64))
    q2 = q.copy()
    q2[1, 2, 5], q2[2, 0, 1] = np.nan, np.inf
    got = run(q2, q2, [1, 2, 3], np.ones(64, np.float32), None, rotary_frequencies(1e4, 64))
    assert np.isnan(got[0][1, 2]).all()
    for g, c in zip(got, clean):
        g[1, 2], g[2, 0] = c[1, 2], c[2, 0]
        np.testing.assert_array_equal(g, c)


def test_captured():
    rng = np.random.default_rng(8)
    stream = Stream()
    q = rng.normal(size=(5, 4, 64)).astype(np.float32)
    freq = rotary_frequencies(1e4, 32)
    d, out, pos, df = upload(q), DeviceArray.from_host(np.zeros_like(q)), upload(np.arange(5), np.int32), upload(freq, np.float64)
    rotate_heads(d, None, 4, 0, 64, 5, pos, df, 32, d_q_out=out, stream=stream)
    with Graph.capture(stream) as g:
        rotate_heads(d, None, 4, 0, 64, 5, pos, df, 32, d_q_out=out, stream=stream)
    for step in range(3):
        positions = np.arange(5) * 100 + step
        pos.upload(positions.astype(np.int32))
        synchronize()
        g.launch(stream)
        synchronize()
        want, tol = heads_of(q, positions, None, freq, 1e-6)
        assert (np.abs(out.to_host(np.float32, q.shape) - want) <= tol).all()
    g.close()


def test_refused_on_the_device_too():
    with DeviceArray(4096) as d:
        with pytest.raises(GpuError, match="rotary"):
            rotate_heads(d, d, 1, 1, 64, 1, d, d, 63)
        with pytest.raises(GpuError, match="stride"):
            rotate_heads(d, d, 2, 1, 64, 1, d, d, 64, q_stride=64)
