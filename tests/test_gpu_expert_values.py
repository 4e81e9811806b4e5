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


def _kind(got, want):
    """NaN where want is, infinities where want has them and of their sign; finite elsewhere."""
    inf = np.isinf(want)
    return (np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), inf) and
            np.array_equal(np.sign(got[inf]), np.sign(want[inf])))


@pytest.mark.parametrize("xdtype", [W.F32, W.F16, W.BF16])
@pytest.mark.parametrize("fmt", [W.MXFP4, W.BF16])
@pytest.mark.parametrize("n,gate", [(3, False), (3, True), (300, False), (300, True)])
def test_infinities_in_the_matrix(hip, dev, fmt, xdtype, n, gate):
    """Infinities in a matrix (MXFP4: values past fp32's) give what fp32 products and sums give: infinities of either
    sign, NaN from two of them or from zeros of x; other outputs, unnamed rows and other groups' rows are as without."""
    rng = np.random.default_rng(n)
    experts, rows, cols = 3, 70, 160
    raws, ws = [], []
    for phase in range(2 if gate else 1):
        if fmt == W.MXFP4:
            codes, scales = random_mx(rng, experts * rows, cols)
            for r, block, s, c in ((5, 0, 254, 7), (5 + rows, 1, 254, 12), (9 + rows, 4, 253, 6), (11, 2, 254, 4), (20, 0, 254, 7)):
                r += phase  # a pair's gate and up rows beside each other
                scales[r, block] = s
                codes[r, block * 32:block * 32 + 32] = 0
                codes[r, block * 32 + 7] = c
            codes[20 + phase, 8] = 15  # -6 beside 6
            scales[30, 1], codes[30, 32:64] = 253, 5  # 3 * 2^126 is finite
            codes[30, 33:64] = 0
            raws.append(W.encode_mxfp4(codes, scales))
            w = mx_values(codes, scales)
        else:
            bits, w = encode(W.BF16, rng.standard_normal((experts * rows, cols)) * 0.02)
            for r, k, v in ((5, 7, np.inf), (5 + rows, 39, -np.inf), (9 + rows, 135, np.inf), (20, 7, np.inf), (20, 8, -np.inf)):
                w[r + phase, k] = v
                bits[r + phase, k] = 0x7f80 if v > 0 else 0xff80
            raws.append(bits.reshape(-1).view(np.uint8))
        with np.errstate(over="ignore"):
            ws.append(w.astype(np.float32).astype(np.float64).reshape(experts, rows, cols))
    x = rng.standard_normal((n, cols))
    x[0, 7] = 0  # times an infinity: NaN
    if n > 2:
        x[2, 39] = -0.0
    bits, x = encode(xdtype, x)
    counts = [1, 0, 2] if n == 3 else [120, 90, 80]
    m = sum(counts)
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    index = rng.permutation(n).astype(np.int32)
    index[m - 1] = -1
    e = hip.Experts(fmt, experts, rows, cols, *raws)
    out = dev.put(np.full((n, rows), 7, np.float32))
    e.mul_device(xdtype, dev.put(bits), 0, cols, n, dev.put(offsets), dev.put(index), n, W.F32, out, rows)
    got = dev.get(out, (n, rows))
    e.close()
    assert (got[m:] == 7).all() and (got[m - 1] == 0).all()
    with np.errstate(all="ignore"):
        for i in range(experts):
            for r in range(offsets[i], min(offsets[i + 1], m - 1)):
                # (the sums are fp32: those past its range are infinities before the gate sees them)
                y = [(x[index[r]] * w[i]).sum(1) for w in ws]
                y = [np.where(np.abs(v) > 3.41e38, np.sign(v) * np.inf, v) for v in y]
                want = silu(y[0]) * y[1] if gate else y[0]
                want = np.where(np.abs(want) > 3.41e38, np.sign(want) * np.inf, want)
                assert _kind(got[r], want), (i, r)
                ok = np.isfinite(want)
                if gate:
                    assert np.all(np.abs(got[r] - want)[ok] <= 1e-4 * (np.abs(want[ok]) + np.abs(y[1][ok])) + 1e-4)
                else:
                    tol = (cols + 128) * 2.0 ** -24 * (np.abs(x[index[r]]) * np.abs(ws[0][i])).sum(1)
                    assert np.all((np.abs(got[r] - want) <= tol)[ok])


@pytest.mark.parametrize("n", [4, 200])
@pytest.mark.parametrize("fmt", [W.MXFP4, W.BF16])
def test_smallest_values(hip, dev, fmt, n):
    """fp32 rows down to subnormal values keep their bits from 2^-133 up (bf16's smallest number, of their last plane)."""
    rng = np.random.default_rng(n)
    rows, cols = 40, 256
    if fmt == W.MXFP4:
        codes, scales = random_mx(rng, rows, cols, 215, 225)
        raw, w = W.encode_mxfp4(codes, scales), mx_values(codes, scales)
    else:
        bits, w = encode(W.BF16, rng.standard_normal((rows, cols)) * 2.0 ** 95)
        raw = bits.reshape(-1).view(np.uint8)
    x = (rng.standard_normal((n, cols)) * 2.0 ** -rng.integers(105, 135, (n, 1))).astype(np.float32)
    e = hip.Experts(fmt, 1, rows, cols, raw)
    out = dev.put(np.zeros((n, rows), np.float32))
    e.mul_device(W.F32, dev.put(x), 0, cols, n, dev.put(np.array([0, n], np.int32)), 0, n, W.F32, out, rows)
    got = dev.get(out, (n, rows))
    e.close()
    x = x.astype(np.float64)
    tol = (cols + 128) * 2.0 ** -24 * (np.abs(x) @ np.abs(w).T) + 2.0 ** -133 * np.abs(w).sum(1)
    assert np.all(np.abs(got - x @ w.T) <= tol)


@pytest.mark.parametrize("n,rows,cols", [(131072, 40, 32), (2080, 100, 2016), (32767, 20, 128), (43690, 36, 96)])
def test_largest_products_without_allocation(hip, dev, n, rows, cols):
    """MXFP4 weights with as many rows as the no-allocation array holds (n * cols up to 2^22; at 32 columns the planes
    fill it, at 2016 the parts' sums lie behind them): the same bits as with allocation."""
    rng = np.random.default_rng(cols)
    raw, _ = matrices(rng, W.MXFP4, 1, rows, cols)
    w = hip.Weight(W.Tensor(W.MXFP4, rows, cols, raw))
    x, out = dev.put(rng.standard_normal((n, cols)).astype(np.float32)), dev.put(np.full((n, rows), np.nan, np.float32))
    w.mul_device(x, n, out)
    want = dev.get(out, (n, rows)).copy()
    assert np.isfinite(want).all() and want.std() > 0
    dev.fill(out, np.full((n, rows), np.nan, np.float32))
    w.mul_device_noalloc(x, n, out)
    assert np.array_equal(dev.get(out, (n, rows)), want)
    w.close()
