"""Values of the expert products where their arithmetic could go wrong, on the GPU against float64."""
import numpy as np
import pytest

from experts_fixture import Device, encode, matrices, mx_rows, mx_values, random_mx, silu
from tinyoai_amd import weights as W

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    from tinyoai_amd import hip as H
    H.lib()
    return H


@pytest.fixture
def dev():
    d = Device()
    yield d
    d.close()


@pytest.mark.parametrize("few", [True, False])
def test_gate_values(hip, dev, few):
    """silu(g) * u for gates over the whole of fp32, most of them about -88, where 1 + e^-g passes 2^126 (its reciprocal
    is subnormal) and 2^128. The sums are exact (a gate is x's first column, u a power of two), so what is left is the
    gate itself: 2^t and the reciprocal (a unit in the last place each), five roundings, all relative; and a rounding of
    silu below fp32's normal numbers, in units of 2^-149."""
    ups = 2.0 ** np.array([0, 60, 100, 120])
    g = np.concatenate([np.linspace(-110, 110, 600), np.linspace(-89.5, -86.5, 400), -(2.0 ** np.arange(-30, 128)),
                        2.0 ** np.arange(-30, 8), [0.0, -87.336545, -88.72284, -3.4e38]]).astype(np.float32)
    rows, cols = len(ups), 32
    gate, up = np.zeros((rows, cols)), np.zeros((rows, cols))
    gate[:, 0], up[:, 1] = 1, ups
    e = hip.Experts(W.BF16, 1, rows, cols, *(encode(W.BF16, m)[0].reshape(-1).view(np.uint8) for m in (gate, up)))
    x = np.zeros((len(g), cols), np.float32)
    x[:, 0], x[:, 1] = g, 1
    px, out = dev.put(x), dev.put(np.zeros((len(g), rows), np.float32))
    step = 4 if few else len(g)  # rows of a call
    for i in range(0, len(g), step):
        n = min(step, len(g) - i)
        e.mul_device(W.F32, px + i * cols * 4, 0, cols, n, dev.put(np.array([0, n], np.int32)), 0, n, W.F32,
                     out + i * rows * 4, rows)
    got = dev.get(out, (len(g), rows)).astype(np.float64)
    e.close()
    s = silu(g.astype(np.float64))[:, None]
    want = s * ups
    big = np.abs(want) > 3.4e38
    tol = 10 * 2.0 ** -24 * np.abs(want) + 2.0 ** -149 * (ups + 1)
    assert np.all((np.abs(got - want) <= tol) | big), g[np.any((np.abs(got - want) > tol) & ~big, 1)]
    assert np.all(np.isinf(got[big]) & (got[big] > 0))


LONG = [(W.MXFP4, W.F32, 70, 96, 65536), (W.MXFP4, W.F32, 1024, 4096, 16384), (W.MXFP4, W.F32, 1024, 1664, 16384),
        (W.MXFP4, W.F16, 1024, 4096, 16384), (W.MXFP4, W.BF16, 1024, 1664, 32768), (W.MXFP4, W.MXFP4, 1024, 4096, 131072),
        (W.BF16, W.F32, 64, 64, 65536), (W.BF16, W.F32, 2048, 3328, 8192), (W.BF16, W.F16, 1024, 4096, 16384),
        (W.BF16, W.BF16, 2048, 3328, 32768), (W.BF16, W.BF16, 4096, 3584, 20480), (W.BF16, W.F32, 3, 20, 1 << 22)]


@pytest.mark.parametrize("fmt,xdtype,n,rows,cols", LONG)
def test_long_rows(hip, dev, fmt, xdtype, n, rows, cols):
    """Products of long rows round no more than fp32 sums of 512 columns in float64 totals do, as the framework's other
    products of fp32 rows (in the norm, as of a random walk: a quarter of sqrt(512) half-ulps of the sum's final size,
    with a margin of a half). A run of 1024 columns rounds at every 16 of each of three planes at most, 192 times, and
    its totals 320 times up to 2^18 columns; past those the totals are doubles. The rows repeat 64 of x and 20 or 32 of
    the matrix."""
    rng = np.random.default_rng(n + cols)
    few = 20 if rows == 20 else 32
    raw, w = matrices(rng, fmt, 1, few, cols)
    raw = np.tile(raw.reshape(few, -1), (rows // few, 1)).reshape(-1)
    at = np.arange(n) % 64
    ps = 0
    if xdtype == W.MXFP4:
        q = random_mx(rng, 64, cols, 120, 130)
        x = mx_values(*q)
        px, ps = (dev.put(a) for a in mx_rows(*(a[at] for a in q)))
    else:
        bits, x = encode(xdtype, rng.standard_normal((min(n, 64), cols)))
        px = dev.put(bits[at])
    out = dev.put(np.full((n, rows), np.nan, np.float32))
    want = (x @ w[0].T)[at]

    def check():
        got = dev.get(out, (n, rows)).astype(np.float64)
        err = np.linalg.norm(got.reshape(n, -1, few) - want[:, None], axis=(0, 2)) / np.linalg.norm(want)
        assert err.max() <= 1.5 * 0.25 * np.sqrt(512.0) * 2.0 ** -24

    e = hip.Experts(fmt, 1, rows, cols, raw)
    e.mul_device(xdtype, px, ps, cols, n, dev.put(np.array([0, n], np.int32)), 0, n, W.F32, out, rows)
    check()
    e.close()
    if fmt == W.MXFP4 and xdtype in (W.F32, W.MXFP4):
        g = hip.Weight(W.Tensor(fmt, rows, cols, raw))
        dev.fill(out, np.full((n, rows), np.nan, np.float32))
        g.mul_device(px, n, out) if not ps else g.mul_mxfp4_device(px, ps, n, out)
        check()
        g.close()
