"""The mixture-of-experts operators on the GPU against float64: MXFP4 rows,
products of MXFP4 and BF16 matrices grouped by expert, routing and the sum of
the experts' rows."""
import ctypes as C

import numpy as np
import pytest

from experts_fixture import (EPS, WIDTH, Device, bits_dtype, decode, encode, matrices, mx_quantize, mx_rows, mx_values,
                             random_mx, silu)
from tinyoai_amd import weights as W

pytestmark = pytest.mark.gpu

TYPES = (W.F32, W.F16, W.BF16)


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


# ---------------------------------------------------------------- MXFP4 rows
def _edge_rows(rng, n, cols, dtype):
    """Rows over the type's whole range: halfway values, subnormals, zeros, the largest values, outliers."""
    x = rng.standard_normal((n, cols)).astype(np.float32)
    if n == 1:
        return x
    x *= np.float32(2.0) ** rng.integers(-12, 12, (n, 1)).astype(np.float32)
    x[0, :32] = np.float32(2.0) ** rng.integers(-3, 3) * rng.choice([.25, .75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7], 32)
    x[1, :32] = 0
    x[1, 32:64] = -0.0
    if dtype != W.F16:
        x[2] *= np.float32(1e-38)
        x[3, :32] = rng.choice([1.4e-45, 5.9e-39, -1.2e-38, 2e-39], 32)
        x[4, ::5] = 3.3e38
    else:
        x[2] *= np.float32(6e-8)
        x[4, ::5] = 65504
    x[5, 7] *= 1e4 if dtype != W.F16 else 10
    return x


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,cols,pad,shift", [(1, 32, 0, 0), (7, 64, 0, 0), (9, 160, 1, 0), (33, 256, 32, 4),
                                              (300, 2560, 0, 0), (6, 6912, 3, 0)])
def test_quantize(hip, dev, dtype, n, cols, pad, shift):
    """Codes, scales and the values they stand for, bit for bit; padding is written as zeros; other values of wider rows
    are not touched."""
    rng = np.random.default_rng(n * cols)
    bits, x = encode(dtype, _edge_rows(rng, n, cols + pad, dtype))
    codes, scales = mx_quantize(x[:, :cols])
    want_c, want_s = mx_rows(codes, scales)
    px = dev.put(bits, shift)
    pc, ps = dev.put(np.full_like(want_c, 0xEE)), dev.put(np.full_like(want_s, 0xEE))
    hip.quantize_mxfp4(dtype, px, cols + pad, n, cols, pc, ps)
    got_c, got_s = dev.get(pc, want_c.shape, np.uint8), dev.get(ps, want_s.shape, np.uint8)
    assert np.array_equal(got_s, want_s)
    assert np.array_equal(got_c, want_c)
    values = mx_values(codes, scales)
    for odtype in TYPES:
        out = dev.put(np.full((n, cols + pad), 7, bits_dtype(odtype)), shift)
        hip.dequantize_mxfp4(pc, ps, n, cols, odtype, out, cols + pad)
        raw = dev.get(out, (n, cols + pad), bits_dtype(odtype))
        got = decode(odtype, raw)[:, :cols]
        with np.errstate(over="ignore"):
            want = values.astype(np.float16).astype(np.float64) if odtype == W.F16 else values
        assert np.array_equal(got, want)
        assert (raw[:, cols:] == 7).all()


def test_quantize_not_finite(hip, dev):
    """A block with an infinity or NaN is NaN; its neighbours are not."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((3, 256)).astype(np.float32)
    x[0, 40], x[1, 0], x[2, 255] = np.inf, np.nan, -np.inf
    units = 2
    px, pc, ps = dev.put(x), dev.put(np.zeros((3, 64 * units), np.uint8)), dev.put(np.zeros((3, 4 * units), np.uint8))
    out = dev.put(np.zeros((3, 256), np.float32))
    hip.quantize_mxfp4(W.F32, px, 256, 3, 256, pc, ps)
    hip.dequantize_mxfp4(pc, ps, 3, 256, W.F32, out, 256)
    got = dev.get(out, (3, 256))
    bad = np.zeros((3, 8), bool)
    bad[0, 1] = bad[1, 0] = bad[2, 7] = True
    assert np.array_equal(np.isnan(got).reshape(3, 8, 32), np.broadcast_to(bad[..., None], (3, 8, 32)))
    with np.errstate(invalid="ignore"):
        want = mx_values(*mx_quantize(x.astype(np.float64)))
    assert np.array_equal(got[~np.isnan(got)], want[~np.isnan(want)])


# ---------------------------------------------------------------- products
def _x_rows(rng, dev, xdtype, n, cols, pad=0, shift=0):
    """(pointer, scales pointer, float64 values) of n rows."""
    if xdtype == W.MXFP4:
        q = random_mx(rng, n, cols, 120, 130)
        c, s = mx_rows(*q)
        return dev.put(c), dev.put(s), mx_values(*q)
    x = rng.standard_normal((n, cols + pad)) * np.exp(rng.standard_normal(cols + pad))
    if n > 2:
        x *= 2.0 ** rng.integers(-6, 6, (n, 1))
    bits, v = encode(xdtype, x)
    return dev.put(bits, shift), 0, v[:, :cols]


def _tolerance(x, w, cols):
    """Every product is exact in fp32 (planes of 8 bits times 8 or 2 bits; fp32 multiply-adds round once with their
    sum); at most 3 * cols / 8 + 64 sums on the matrix cores, each off by 2^-23 of the partial sum at most, or cols
    sums off by 2^-24."""
    return (cols + 128) * 2.0 ** -24 * (np.abs(x) @ np.abs(w).T) + 1e-44


def _expected(x, ws, gate, odtype, cols):
    """(float64 result, bound of the error) of rows x with one expert's matrices."""
    y, t = x @ ws[0].T, _tolerance(x, ws[0], cols)
    if gate:
        u, tu = x @ ws[1].T, _tolerance(x, ws[1], cols)
        s = silu(y)
        # |silu'| < 1.1; the gate's own exp, sum, quotient and product: 8 roundings
        t = 1.1 * t * (np.abs(u) + tu) + np.abs(s) * tu + 8 * 2.0 ** -24 * np.abs(s * u)
        y = s * u
    return y, t + EPS[odtype] * (np.abs(y) + t) + (2.0 ** -25 if odtype == W.F16 else 1e-44)


def _close(got, want, tol, odtype):
    """Within tol; values from 65520 on (half a step past fp16's largest, 65504) round to an infinity in fp16."""
    ok = np.abs(got - want) <= tol
    return ok | (np.isinf(got) & (got * want > 0) & (np.abs(want) + tol >= 65520)) if odtype == W.F16 else ok


SHAPES = [(1, 1, 32), (3, 2, 96), (2, 15, 128), (16, 16, 160), (17, 33, 256), (31, 64, 512), (40, 300, 1024), (5, 70, 2560),
          (129, 257, 288), (300, 130, 672), (1000, 20, 64), (2, 6912, 2560), (1, 2560, 6912), (48, 260, 2560), (33, 1001, 4160),
          (12, 130, 6912), (200, 90, 4096), (65, 7, 12800)]


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("n,rows,cols", SHAPES)
def test_weight_product(hip, dev, n, rows, cols, quantised):
    """An MXFP4 weight times fp32 and times MXFP4 rows; mul, mul_device and mul_device_noalloc give the same bits."""
    rng = np.random.default_rng(n + rows + cols)
    raw, w = matrices(rng, W.MXFP4, 1, rows, cols)
    g = hip.Weight(W.Tensor(W.MXFP4, rows, cols, raw))
    assert np.array_equal(g.read_values(0, rows * cols).reshape(rows, cols), w[0].astype(np.float32))
    out = dev.put(np.full((n, rows), np.nan, np.float32))
    px, ps, x = _x_rows(rng, dev, W.MXFP4 if quantised else W.F32, n, cols)
    if quantised:
        g.mul_mxfp4_device(px, ps, n, out)
    else:
        g.mul_device(px, n, out)
    got = dev.get(out, (n, rows))
    want, tol = _expected(x, w, False, W.F32, cols)
    assert np.all(np.abs(got - want) <= tol)
    if not quantised:
        out2 = dev.put(np.full((n, rows), np.nan, np.float32))
        g.mul_device_noalloc(px, n, out2)
        assert np.array_equal(dev.get(out2, (n, rows)), got)
        assert np.array_equal(g.mul(x.astype(np.float32)), got)
    g.close()


def _grouped(hip, dev, seed, fmt, xdtype, counts, rows, cols, gate, odtype, gather, pad=0, shift=0, tail=3):
    """One product grouped by expert, every output and every untouched value checked."""
    rng = np.random.default_rng(seed)
    experts, m = len(counts), int(sum(counts))
    n = m + tail  # rows behind the last group
    data = [matrices(rng, fmt, experts, rows, cols) for _ in range(2 if gate else 1)]
    e = hip.Experts(fmt, experts, rows, cols, *(d[0] for d in data))
    x_rows = max(1, m // 2 + 1) if gather else n
    px, ps, x = _x_rows(rng, dev, xdtype, x_rows, cols, pad, shift)
    index = rng.integers(0, x_rows, n).astype(np.int32)
    if gather and m > 2:
        index[[0, m // 2]] = [-1, x_rows]  # no row
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    ldo = rows + pad
    fresh = np.full((n, ldo), 7, bits_dtype(odtype))
    out = dev.put(fresh, shift)
    po = dev.put(offsets)
    pi = dev.put(index) if gather else 0
    e.mul_device(xdtype, px, ps, cols if xdtype == W.MXFP4 else cols + pad, x_rows, po, pi, n, odtype, out, ldo)
    raw = dev.get(out, (n, ldo), bits_dtype(odtype))
    got = decode(odtype, raw)[:, :rows]
    assert np.array_equal(raw[:, rows:], fresh[:, rows:])
    assert np.array_equal(raw[m:], fresh[m:])
    src = index if gather else np.arange(n)
    xs = np.where(((src >= 0) & (src < x_rows))[:, None], x[np.clip(src, 0, x_rows - 1)], 0)
    for i in range(experts):
        r = slice(offsets[i], offsets[i + 1])
        want, tol = _expected(xs[r], [d[1][i] for d in data], gate, odtype, cols)
        assert np.all(_close(got[r], want, tol, odtype)), (i, np.max(np.abs(got[r] - want) / tol))
    # again on the same handle: the same bits
    dev.fill(out, fresh)
    e.mul_device(xdtype, px, ps, cols if xdtype == W.MXFP4 else cols + pad, x_rows, po, pi, n, odtype, out, ldo)
    assert np.array_equal(dev.get(out, (n, ldo), bits_dtype(odtype)), raw)
    e.close()


COUNTS = {"one": [1], "few": [1, 0, 2, 3, 0, 5, 1, 0], "uneven": [0, 17, 1, 0, 40, 16, 0], "many": [130, 0, 70, 1, 257],
          "empty": [0, 0, 0], "last": [0, 0, 0, 4]}
PAIRS = [(W.MXFP4, W.F32), (W.MXFP4, W.F16), (W.MXFP4, W.BF16), (W.MXFP4, W.MXFP4), (W.BF16, W.F32), (W.BF16, W.F16),
         (W.BF16, W.BF16)]


@pytest.mark.parametrize("fmt,xdtype", PAIRS)
@pytest.mark.parametrize("counts", sorted(COUNTS))
@pytest.mark.parametrize("rows,cols,gate,odtype", [(70, 160, True, W.F32), (33, 96, False, W.BF16),
                                                   (130, 512, True, W.F16), (16, 64, False, W.F32)])
def test_grouped_product(hip, dev, fmt, xdtype, counts, rows, cols, gate, odtype):
    _grouped(hip, dev, rows, fmt, xdtype, COUNTS[counts], rows, cols, gate, odtype, gather=gate)


@pytest.mark.parametrize("fmt,xdtype", PAIRS)
@pytest.mark.parametrize("cols", [32, 2560])
@pytest.mark.parametrize("counts", [[3, 1, 9], [80, 5, 200]])
def test_grouped_product_strides(hip, dev, fmt, xdtype, cols, counts):
    """Wider rows on odd addresses, in and out, with and without an index."""
    for gather, pad, shift in ((True, 3, 4), (False, 8, 16), (False, 1, 2 if xdtype in (W.F16, W.BF16) else 4)):
        odtype = W.F32 if shift == 4 else W.BF16
        _grouped(hip, dev, cols + pad, fmt, xdtype, counts, 50, cols, True, odtype, gather, pad, shift)


@pytest.mark.parametrize("xdtype", TYPES)
@pytest.mark.parametrize("cols", [1, 7, 63, 65, 200, 515])
def test_grouped_bf16_any_columns(hip, dev, xdtype, cols):
    """BF16 matrices have rows of any length."""
    _grouped(hip, dev, cols, W.BF16, xdtype, [2, 0, 19], 37, cols, True, W.F32, True)
    _grouped(hip, dev, cols, W.BF16, xdtype, [200, 90], 37, cols, False, W.F32, False)


@pytest.mark.parametrize("fmt,xdtype", PAIRS)
def test_grouped_many_experts(hip, dev, fmt, xdtype):
    """More experts than a wave has lanes, one of them with most rows."""
    rng = np.random.default_rng(3)
    counts = rng.integers(0, 3, 150)
    counts[140] = 300
    _grouped(hip, dev, 9, fmt, xdtype, counts.tolist(), 20, 128, False, W.F32, True)


@pytest.mark.parametrize("fmt,xdtype", [(W.MXFP4, W.F32), (W.MXFP4, W.MXFP4), (W.BF16, W.BF16)])
def test_grouped_product_offsets(hip, dev, fmt, xdtype):
    """Offsets that fall or leave [0, n] count as the nearest that do not; rows of no group stay."""
    rng = np.random.default_rng(1)
    rows, cols, n = 40, 128, 24
    raw, w = matrices(rng, fmt, 4, rows, cols)
    e = hip.Experts(fmt, 4, rows, cols, raw)
    px, ps, x = _x_rows(rng, dev, xdtype, n, cols)
    for offsets, groups in (([-5, 4, 4, 20, 99], [(0, 4), (4, 4), (4, 20), (20, 24)]),
                            ([2, 8, 5, 9, 9], [(2, 8), (8, 8), (5, 9), (9, 9)]), ([7] * 5, [])):
        out = dev.put(np.full((n, rows), 7, np.float32))
        e.mul_device(xdtype, px, ps, cols, n, dev.put(np.array(offsets, np.int32)), 0, n, W.F32, out, rows)
        got = dev.get(out, (n, rows))
        seen = np.zeros(n, bool)
        allowed = [[] for _ in range(n)]
        for i, (a, b) in enumerate(groups):
            seen[a:b] = True
            for r in range(a, b):
                allowed[r].append(i)
        assert (got[~seen] == 7).all()
        for r in np.nonzero(seen)[0]:  # each output of a row of two groups is either's (both write it, in any order)
            ok = [np.abs(got[r] - x[r] @ w[i].T) <= _tolerance(x[r:r + 1], w[i], cols)[0] * 2 for i in allowed[r]]
            assert np.all(np.any(ok, 0)), (offsets, r)
    e.close()


@pytest.mark.parametrize("fmt,xdtype", [(W.BF16, W.BF16), (W.BF16, W.F32), (W.MXFP4, W.MXFP4), (W.MXFP4, W.F16)])
def test_longest_rows(hip, dev, fmt, xdtype):
    """Rows of 2^22 columns, the longest taken: a few hundred small whole numbers in zeros, so every sum is exact."""
    rng = np.random.default_rng(2)
    rows, cols, n, offsets = 17, 1 << 22, 3, [0, 2, 3]
    at = np.unique(np.concatenate([[0, 1, 127, 128, cols // 2, cols - 1, cols - 65], rng.integers(0, cols, 200)]))
    codes = np.zeros((2, rows, cols), np.uint8)
    codes[..., at] = rng.choice([0, 2, 4, 5, 6, 7, 10, 12], (2, rows, at.size))  # 0, 1, 2, 3, 4, 6, -1, -2
    table = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6])
    if fmt == W.MXFP4:
        raw = np.concatenate([W.encode_mxfp4(c, np.full((rows, cols // 32), 127, np.uint8)) for c in codes])
    else:
        raw = (table.astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)[codes].reshape(-1).view(np.uint8)
    xc = np.zeros((n, cols), np.uint8)
    xc[:, at] = rng.choice([0, 2, 4, 5, 6, 7, 10, 12], (n, at.size))
    ps = 0
    if xdtype == W.MXFP4:
        c, s = mx_rows(xc, np.full((n, cols // 32), 127, np.uint8))
        px, ps = dev.put(c), dev.put(s)
    else:
        px = dev.put(encode(xdtype, table)[0][xc])
    e = hip.Experts(fmt, 2, rows, cols, raw)
    out = dev.put(np.full((n, rows), np.nan, np.float32))
    e.mul_device(xdtype, px, ps, cols, n, dev.put(np.array(offsets, np.int32)), 0, n, W.F32, out, rows)
    got = dev.get(out, (n, rows))
    e.close()
    for i in range(2):
        r = slice(offsets[i], offsets[i + 1])
        assert np.array_equal(got[r], table[xc[r]][:, at] @ table[codes[i][:, at]].T)


@pytest.mark.parametrize("counts", [[1, 0, 4], [40, 0, 90, 33]])
@pytest.mark.parametrize("fmt,xdtype", PAIRS)
def test_gathered_from_many_rows(hip, dev, fmt, xdtype, counts):
    """An index into far more rows than it names, up to the last ones of more than 4 GiB."""
    rng = np.random.default_rng(len(counts))
    rows, cols, n, m = 40, 256, sum(counts) + 2, sum(counts)
    raw, w = matrices(rng, fmt, len(counts), rows, cols)
    e = hip.Experts(fmt, len(counts), rows, cols, raw)
    unit = 64 if xdtype == W.MXFP4 else WIDTH[xdtype] * cols  # MXFP4: of a row's 128 columns, a unit after the other
    x_rows = (1 << 32) // (unit * (2 if xdtype == W.MXFP4 else 1)) + 1000
    if xdtype == W.MXFP4:
        x_rows = min(x_rows, 1 << 25)
    src = np.sort(rng.choice(x_rows - 1, n - 1, False))
    src = np.append(src, x_rows - 1)[rng.permutation(n)].astype(np.int32)
    px, ps = dev.room(x_rows * unit * (2 if xdtype == W.MXFP4 else 1)), 0
    if xdtype == W.MXFP4:
        ps = dev.room(x_rows * 8)
        q = random_mx(rng, n, cols, 120, 130)
        c, s = mx_rows(*q)
        x = mx_values(*q)
        for i, r in enumerate(src):
            for u in range(2):
                dev.fill(px + (u * x_rows + int(r)) * 64, c[u, i])
                dev.fill(ps + (u * x_rows + int(r)) * 4, s[u, i])
    else:
        bits, x = encode(xdtype, rng.standard_normal((n, cols)))
        for i, r in enumerate(src):
            dev.fill(px + int(r) * unit, bits[i])
    out = dev.put(np.full((n, rows), 7, np.float32))
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    e.mul_device(xdtype, px, ps, cols, x_rows, dev.put(offsets), dev.put(src), n, W.F32, out, rows)
    got = dev.get(out, (n, rows))
    assert (got[m:] == 7).all()
    for i in range(len(counts)):
        r = slice(offsets[i], offsets[i + 1])
        want, tol = _expected(x[r], w[i:i + 1], False, W.F32, cols)
        assert np.all(np.abs(got[r] - want) <= tol), i
    e.close()


@pytest.mark.parametrize("n", [1, 5, 40, 200])
@pytest.mark.parametrize("fmt,xdtype", [(W.MXFP4, W.F32), (W.MXFP4, W.MXFP4), (W.BF16, W.F32), (W.BF16, W.BF16)])
def test_product_extreme_values(hip, dev, fmt, xdtype, n):
    """Very large and small values keep their bits; an infinity or NaN of x reaches its own row only, one of the matrix
    its own outputs only."""
    rng = np.random.default_rng(n)
    rows, cols = 40, 256
    if fmt == W.MXFP4:
        codes, scales = random_mx(rng, rows, cols)
        scales[3], scales[4] = 240, 3
        scales[5, 2] = 255
        raw, w = W.encode_mxfp4(codes, scales), mx_values(codes, scales)
    else:
        v = rng.standard_normal((rows, cols)) * 0.02
        v[3] *= 2.0 ** 110
        v[4] *= 2.0 ** -110
        bits, w = encode(W.BF16, v)
        bits[5, 70] = 0x7fc0
        w[5, 70] = np.nan
        raw = bits.reshape(-1).view(np.uint8)
    e = hip.Experts(fmt, 1, rows, cols, raw)
    if xdtype == W.MXFP4:
        xc, xs = random_mx(rng, n, cols, 120, 130)
        if n > 2:
            xs[0], xs[1] = 20, 100
            xs[2, 1] = 255
        c, s = mx_rows(xc, xs)
        px, ps, x = dev.put(c), dev.put(s), mx_values(xc, xs)
    else:
        x = rng.standard_normal((n, cols)).astype(np.float32)
        if n > 2:
            x[0] *= np.float32(2.0 ** -100)
            x[1] *= np.float32(2.0 ** -20)
            x[2, 33] = np.inf
        if n > 4:
            x[3, 200] = np.nan
            x[4, 0] = -np.inf
        finite = np.isfinite(x)
        bits, v = encode(xdtype, np.where(finite, x, 0))
        if xdtype == W.F32:
            px = dev.put(x)
        else:
            bits[~finite] = (x[~finite].view(np.uint32) >> 16).astype(np.uint16)
            px = dev.put(bits)
        ps, x = 0, np.where(finite, v, x.astype(np.float64))
    out = dev.put(np.zeros((n, rows), np.float32))
    e.mul_device(xdtype, px, ps, cols, n, dev.put(np.array([0, n], np.int32)), 0, n, W.F32, out, rows)
    got = dev.get(out, (n, rows)).astype(np.float64)
    e.close()
    with np.errstate(all="ignore"):
        fx, fw = np.isfinite(x).all(1), np.isfinite(w).all(1)
        want, tol = _expected(np.where(np.isfinite(x), x, 0), [np.where(np.isfinite(w), w, 0)], False, W.F32, cols)
        ok = np.outer(fx, fw)
        # what fp32 cannot hold becomes infinite; below its normal numbers sums lose bits (2^-149 a step, 2^-126 a flush)
        big = np.abs(want) > 3.4e38
        small = cols * 2.0 ** -126 * 3
        assert np.all((np.abs(got - want) <= tol + small) | ~ok | big)
        assert not np.isfinite(got[~fx]).any() and not np.isfinite(got[:, ~fw]).any()


@pytest.mark.parametrize("fmt,xdtype,n", [(W.MXFP4, W.F32, 5), (W.MXFP4, W.F32, 300), (W.MXFP4, W.MXFP4, 300),
                                          (W.BF16, W.F16, 90), (W.BF16, W.BF16, 300), (W.MXFP4, W.BF16, 40)])
def test_captured_and_concurrent_products(hip, dev, fmt, xdtype, n):
    """Two graphs captured from one handle and eager calls on a third stream, all in flight together, give an eager
    call's bits on every replay, with eager work between the replays."""
    rng = np.random.default_rng(n)
    rows, cols, experts = 200, 512, 4
    raw, _ = matrices(rng, fmt, experts, rows, cols)
    e = hip.Experts(fmt, experts, rows, cols, raw)
    rt = dev.rt
    streams, execs = [C.c_void_p() for _ in range(3)], []
    xs = [_x_rows(rng, dev, xdtype, n, cols)[:2] for _ in range(3)]
    po = dev.put(np.linspace(0, n, experts + 1).astype(np.int32))
    y = [dev.put(np.zeros((n, rows), np.float32)) for _ in range(4)]

    def call(i, out, stream=0):
        e.mul_device(xdtype, *xs[i], cols, n, po, 0, n, W.F32, out, rows, stream)

    try:
        for st in streams:
            assert rt.hipStreamCreateWithFlags(C.byref(st), 1) == 0
        for i in range(2):
            graph, ex = C.c_void_p(), C.c_void_p()
            assert rt.hipStreamBeginCapture(streams[i], 0) == 0
            call(i, y[i], streams[i].value)
            call(i, y[i], streams[i].value)
            assert rt.hipStreamEndCapture(streams[i], C.byref(graph)) == 0
            assert rt.hipGraphInstantiate(C.byref(ex), graph, None, None, C.c_size_t(0)) == 0
            rt.hipGraphDestroy(graph)
            execs.append(ex)
        want = []
        for i in range(3):
            call(i, y[3])
            want.append(dev.get(y[3], (n, rows)).copy())
        assert np.abs(want[0]).max() > 0
        for _ in range(3):
            for i in range(3):
                dev.fill(y[i], np.zeros((n, rows), np.float32))
            for _ in range(4):
                for i in range(2):
                    assert rt.hipGraphLaunch(execs[i], streams[i]) == 0
                call(2, y[2], streams[2].value)
            for i in range(3):
                assert np.array_equal(dev.get(y[i], (n, rows)), want[i]), i
    finally:
        for ex in execs:
            rt.hipGraphExecDestroy(ex)
        for st in streams:
            rt.hipStreamDestroy(st)
        e.close()


@pytest.mark.parametrize("quantised", [False, True])
def test_captured_weight_product(hip, dev, quantised):
    """A product that is cut over its columns: two captured calls on two streams and eager calls between the replays."""
    rng = np.random.default_rng(4)
    n, rows, cols, rt = 40, 300, 4096, dev.rt
    raw, _ = matrices(rng, W.MXFP4, 1, rows, cols)
    w = hip.Weight(W.Tensor(W.MXFP4, rows, cols, raw))
    xs = [_x_rows(rng, dev, W.MXFP4 if quantised else W.F32, n, cols)[:2] for _ in range(3)]
    y = [dev.put(np.zeros((n, rows), np.float32)) for _ in range(3)]
    streams, execs = [C.c_void_p() for _ in range(2)], []

    def call(i, out, stream=0):
        w.mul_mxfp4_device(*xs[i], n, out, stream) if quantised else w.mul_device(xs[i][0], n, out, stream)

    try:
        for i, st in enumerate(streams):
            graph, ex = C.c_void_p(), C.c_void_p()
            assert rt.hipStreamCreateWithFlags(C.byref(st), 1) == 0
            assert rt.hipStreamBeginCapture(st, 0) == 0
            call(i, y[i], st.value)
            assert rt.hipStreamEndCapture(st, C.byref(graph)) == 0
            assert rt.hipGraphInstantiate(C.byref(ex), graph, None, None, C.c_size_t(0)) == 0
            rt.hipGraphDestroy(graph)
            execs.append(ex)
        want = []
        for i in range(3):
            call(i, y[2])
            want.append(dev.get(y[2], (n, rows)).copy())
        assert np.abs(want[0]).max() > 0
        for _ in range(3):
            for i in range(3):
                dev.fill(y[i], np.zeros((n, rows), np.float32))
            for _ in range(3):
                for i in range(2):
                    assert rt.hipGraphLaunch(execs[i], streams[i]) == 0
                call(2, y[2])
            for i in range(3):
                assert np.array_equal(dev.get(y[i], (n, rows)), want[i]), i
    finally:
        for ex in execs:
            rt.hipGraphExecDestroy(ex)
        for st in streams:
            rt.hipStreamDestroy(st)
        w.close()


def test_two_threads(hip, dev):
    """Calls of two threads on one handle, each on its own stream: every call's bits are an idle handle's."""
    import threading
    rng = np.random.default_rng(6)
    rows, cols, experts, n = 100, 256, 4, 120
    raw, _ = matrices(rng, W.MXFP4, experts, rows, cols)
    e = hip.Experts(W.MXFP4, experts, rows, cols, raw)
    po = dev.put(np.linspace(0, n, experts + 1).astype(np.int32))
    xs = [_x_rows(rng, dev, W.F32, n, cols)[0] for _ in range(2)]
    y = [[dev.put(np.zeros((n, rows), np.float32)) for _ in range(10)] for _ in range(2)]
    streams, errors = [C.c_void_p() for _ in range(2)], []
    for st in streams:
        assert dev.rt.hipStreamCreateWithFlags(C.byref(st), 1) == 0

    def work(i):
        try:
            for out in y[i]:
                e.mul_device(W.F32, xs[i], 0, cols, n, po, 0, n, W.F32, out, rows, streams[i].value)
        except Exception as err:
            errors.append(err)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    got = [[dev.get(out, (n, rows)).copy() for out in outs] for outs in y]
    for i in range(2):
        e.mul_device(W.F32, xs[i], 0, cols, n, po, 0, n, W.F32, y[i][0], rows)
        want = dev.get(y[i][0], (n, rows))
        assert np.abs(want).max() > 0 and all(np.array_equal(g, want) for g in got[i])
    for st in streams:
        dev.rt.hipStreamDestroy(st)
    e.close()


def test_refusals_of_handles(hip, dev):
    rng = np.random.default_rng(0)
    raw, _ = matrices(rng, W.BF16, 2, 8, 64)
    e = hip.Experts(W.BF16, 2, 8, 64, raw)
    A = dev.put(np.zeros(4096, np.uint8))

    def call(xd=W.F32, x=A, xs=0, ldx=64, xr=4, off=A, n=4, od=W.F32, out=A, ldo=8, h=e):
        h.mul_device(xd, x, xs, ldx, xr, off, 0, n, od, out, ldo)

    for bad, match in ((dict(xd=W.MXFP4, xs=A), "need MXFP4 experts"), (dict(xd=W.Q8_0), "unsupported x type"),
                       (dict(ldx=63), "63 apart"), (dict(ldo=7), "7 apart"), (dict(xr=3), "without an index"),
                       (dict(n=0), "invalid product"), (dict(off=None), "invalid product"), (dict(out=None), "out is null"),
                       (dict(xs=A), "scales with x"), (dict(x=A + 2), "aligned"), (dict(od=W.Q8_0), "unsupported out")):
        with pytest.raises(hip.TinyoaiError, match=match):
            call(**bad)
    e.close()
    for args, match in (((W.Q8_0, 1, 8, 64, raw[:1]), "unsupported expert tensor type"),
                        ((W.BF16, 2, 8, 64, raw[:-2]), "need 2048 bytes"), ((W.BF16, 0, 8, 64, raw), "invalid matrix shape"),
                        ((W.MXFP4, 1, 8, 48, raw), "whole quant blocks")):
        with pytest.raises(hip.TinyoaiError, match=match):
            hip.Experts(*args)
    raw, _ = matrices(rng, W.MXFP4, 1, 8, 64)
    e = hip.Experts(W.MXFP4, 1, 8, 64, raw)
    with pytest.raises(hip.TinyoaiError, match="rows of 64 values, not 32"):
        call(xd=W.MXFP4, xs=A, ldx=32, h=e)
    with pytest.raises(hip.TinyoaiError, match="16-byte"):
        call(xd=W.MXFP4, x=A + 8, xs=A, h=e)
    with pytest.raises(hip.TinyoaiError, match="invalid MXFP4 rows"):
        call(xd=W.MXFP4, h=e)
    with pytest.raises(hip.TinyoaiError, match="exceeds what one call takes"):  # 2^25 rows' 64 bytes are 2 GiB
        call(xd=W.MXFP4, xs=A, xr=(1 << 25) + 1, n=1 << 20, h=e)
    e.close()
    raw, _ = matrices(rng, W.MXFP4, 1, 130, 64)
    e = hip.Experts(W.MXFP4, 1, 130, 64, raw)  # 2^31 / 32 times 2 tiles of 256 threads
    with pytest.raises(hip.TinyoaiError, match="exceeds what one call takes"):
        call(xr=(1 << 31) - 1, n=(1 << 31) - 1, ldo=130, h=e)
    e.close()
    w = hip.Weight(W.Tensor(W.MXFP4, 130, 64, raw))
    with pytest.raises(hip.TinyoaiError, match="exceeds what one call takes"):
        w.mul_device(A, (1 << 31) - 1, A)
    with pytest.raises(hip.TinyoaiError, match="exceeds what one call takes"):
        w.mul_mxfp4_device(A, A, (1 << 31) - 1, A)
    w.close()
    raw, _ = matrices(rng, W.MXFP4, 1, 8, 64)
    q8 = hip.Weight(W.synthetic_q8_0(8, 64, rng))
    with pytest.raises(hip.TinyoaiError, match="need an MXFP4 weight"):
        q8.mul_mxfp4_device(A, A, 1, A)
    q8.close()
    w = hip.Weight(W.Tensor(W.MXFP4, 8, 64, raw))
    with pytest.raises(hip.TinyoaiError, match="16-byte"):
        w.mul_mxfp4_device(A, A + 1, 1, A)
    with pytest.raises(hip.TinyoaiError, match="no-allocation limit"):
        w.mul_device_noalloc(A, (4 << 20) // 64 + 1, A)
    assert np.array_equal(w.read_values(37, 100), w.read_values(0, 512)[37:137])
    w.close()


# ---------------------------------------------------------------- routing
def _route_expected(x, k, over_all):
    n, experts = x.shape
    ids, weights = np.full((n, k), -1, np.int32), np.zeros((n, k))
    for t in range(n):
        ok = [e for e in range(experts) if x[t, e] > -np.inf]
        best = sorted(ok, key=lambda e: (-x[t, e], e))[:k]
        if not best:
            continue
        m = x[t, best[0]]
        with np.errstate(invalid="ignore"):
            p = np.where(x[t] == m, 1.0, np.exp(x[t] - m))
        weights[t, :len(best)] = p[best] / p[ok if over_all else best].sum()
        ids[t, :len(best)] = best
    flat = ids.reshape(-1)
    order = [s for e in range(experts) for s in np.nonzero(flat == e)[0]]
    tokens, positions = np.full(n * k, -1, np.int32), np.full(n * k, -1, np.int32)
    tokens[:len(order)] = np.array(order, np.int32) // k
    positions[order] = np.arange(len(order))
    offsets = np.concatenate([[0], np.cumsum([(flat == e).sum() for e in range(experts)])]).astype(np.int32)
    return ids, weights, offsets, tokens, positions.reshape(n, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,experts,k,over_all,pad", [(1, 1, 1, False, 0), (1, 8, 8, True, 0), (16, 64, 4, False, 3),
                                                      (32, 65, 8, True, 0), (33, 128, 2, False, 0), (7, 1000, 32, True, 1),
                                                      (500, 200, 5, False, 0), (3000, 7, 3, True, 5), (1500, 512, 1, True, 0),
                                                      (4500, 130, 2, False, 0), (1100, 1024, 8, True, 0), (2, 1024, 32, False, 0),
                                                      (9001, 1, 1, False, 0)])
def test_route(hip, dev, dtype, n, experts, k, over_all, pad):
    """Ties, masked experts (-inf, NaN, every one of a token), infinities and zeros of both signs."""
    rng = np.random.default_rng(n + experts)
    x = (rng.standard_normal((n, experts + pad)) * 1.5).round(1).astype(np.float32)  # many ties
    x[rng.random(x.shape) < 0.1] = -np.inf
    x[rng.random(x.shape) < 0.05] = -0.0
    x[::7, ::3] = 0
    if n > 4:
        x[1] = -np.inf
        x[2, : experts // 2] = np.nan
        x[3, [0, experts - 1]] = np.inf
        x[4] = np.nan
    if dtype == W.BF16:
        finite = np.isfinite(x)
        bits = np.where(finite, encode(W.BF16, np.where(finite, x, 0))[0], (x.view(np.uint32) >> 16).astype(np.uint16))
    else:
        bits = encode(dtype, x)[0]
    v = decode(dtype, np.ascontiguousarray(bits))[:, :experts]
    want = _route_expected(v, k, over_all)
    px = dev.put(bits)
    shapes = [(n, k), (n, k), (experts + 1,), (n * k,), (n, k)]
    types = [np.int32, np.float32, np.int32, np.int32, np.int32]
    p = [dev.put(np.full(s, 99, t)) for s, t in zip(shapes, types)]
    for _ in range(2):
        hip.route(dtype, px, experts + pad, n, experts, k, over_all, *p)
        got = [dev.get(q, s, t) for q, s, t in zip(p, shapes, types)]
        for i in (0, 2, 3, 4):
            assert np.array_equal(got[i], want[i]), i
        # exp, the sum of up to 1000 values (64 lanes of 16, then 6 steps) and the quotient, and the rounding of l - m
        # (at most 2^-24 of 20 in the exponent)
        assert np.all(np.abs(got[1] - want[1]) <= 64 * 2.0 ** -24 * want[1] + 1e-44)


# ---------------------------------------------------------------- combine
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("odtype", TYPES)
@pytest.mark.parametrize("n,k,cols,pad", [(1, 1, 1, 0), (3, 2, 64, 0), (16, 4, 2560, 0), (9, 8, 100, 4), (5, 3, 37, 1),
                                          (700, 5, 260, 0), (6, 3, 515, 0), (4, 2, 259, 2)])
def test_combine(hip, dev, dtype, odtype, n, k, cols, pad):
    rng = np.random.default_rng(n * cols)
    y_rows = max(1, n * k - 1)
    bits, y = encode(dtype, rng.standard_normal((y_rows, cols + pad)))
    pos = rng.integers(0, y_rows, (n, k)).astype(np.int32)
    pos[rng.random((n, k)) < 0.2] = -1
    pos[0, 0] = y_rows if n > 1 else 0
    w = rng.standard_normal((n, k)).astype(np.float32)
    fresh = np.full((n, cols + pad), 7, bits_dtype(odtype))
    out = dev.put(fresh)
    hip.combine(dtype, dev.put(bits), cols + pad, y_rows, dev.put(pos), dev.put(w), n, k, cols, odtype, out, cols + pad)
    raw = dev.get(out, fresh.shape, bits_dtype(odtype))
    ok = (pos >= 0) & (pos < y_rows)
    terms = np.where(ok[..., None], y[np.clip(pos, 0, y_rows - 1)][..., :cols] * w[..., None].astype(np.float64), 0)
    want, mag = terms.sum(1), np.abs(terms).sum(1)
    tol = k * 2.0 ** -24 * mag
    tol = tol + EPS[odtype] * (np.abs(want) + tol) + (2.0 ** -25 if odtype == W.F16 else 1e-44)
    assert np.all(np.abs(decode(odtype, raw)[:, :cols] - want) <= tol)
    assert np.array_equal(raw[:, cols:], fresh[:, cols:])


def test_combine_many_tokens(hip, dev):
    """More tokens than a launch has blocks."""
    rng = np.random.default_rng(8)
    n, rows = (1 << 24) + 3, 50
    y = rng.standard_normal(rows).astype(np.float32)
    pos, w = rng.integers(-1, rows + 1, n).astype(np.int32), rng.random(n, np.float32)
    out = dev.put(np.full(n, 7, np.float32))
    hip.combine(W.F32, dev.put(y), 1, rows, dev.put(pos), dev.put(w), n, 1, 1, W.F32, out, 1)
    want = np.where((pos >= 0) & (pos < rows), y[np.clip(pos, 0, rows - 1)] * w, np.float32(0))
    assert np.array_equal(dev.get(out, n), want)


def test_combine_without_rows(hip, dev):
    """No row at all, and infinities in rows that no position names."""
    y = np.full((4, 8), np.inf, np.float32)
    y[1] = 2
    out = dev.put(np.full((2, 8), 7, np.float32))
    pos = np.array([[-1, -1], [1, -1]], np.int32)
    hip.combine(W.F32, dev.put(y), 8, 4, dev.put(pos), dev.put(np.ones((2, 2), np.float32)), 2, 2, 8, W.F32, out, 8)
    assert dev.get(out, (2, 8)).tolist() == [[0.0] * 8, [2.0] * 8]
    hip.combine(W.F32, dev.put(y), 8, 0, dev.put(pos), dev.put(np.ones((2, 2), np.float32)), 2, 2, 8, W.F32, out, 8)
    assert not dev.get(out, (2, 8)).any()


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("n,experts,k,quantised", [(1, 8, 2, False), (16, 32, 4, False), (16, 32, 4, True), (600, 16, 3, False),
                                                   (600, 16, 3, True)])
def test_expert_layer(hip, dev, n, experts, k, quantised):
    """A layer's experts as they are used: route, gate and up products of the routed tokens, down products, the weighted
    sum; masked logits and a padded token. Captured, replayed with new tokens, each replay against float64."""
    rng = np.random.default_rng(n)
    hidden, inter = 256, 160
    (g_raw, g), (u_raw, u), (d_raw, d) = (matrices(rng, W.MXFP4, experts, *s) for s in
                                          ((inter, hidden), (inter, hidden), (hidden, inter)))
    up, down = hip.Experts(W.MXFP4, experts, inter, hidden, g_raw, u_raw), hip.Experts(W.MXFP4, experts, hidden, inter, d_raw)
    f32, i32, u8 = np.float32, np.int32, np.uint8
    px, pl = dev.put(np.zeros((n, hidden), f32)), dev.put(np.zeros((n, experts), f32))
    ids, wt, off = dev.put(np.zeros((n, k), i32)), dev.put(np.zeros((n, k), f32)), dev.put(np.zeros(experts + 1, i32))
    tok, pos = dev.put(np.zeros(n * k, i32)), dev.put(np.zeros((n, k), i32))
    h, y, out = (dev.put(np.zeros(s, f32)) for s in ((n * k, inter), (n * k, hidden), (n, hidden)))
    (cb, sb), (cb2, sb2) = hip.mxfp4_row_bytes(hidden), hip.mxfp4_row_bytes(inter)
    qc, qs, hc, hs = (dev.put(np.zeros(s, u8)) for s in ((n, cb), (n, sb), (n * k, cb2), (n * k, sb2)))

    def layer(st):
        hip.route(W.F32, pl, experts, n, experts, k, False, ids, wt, off, tok, pos, st)
        if quantised:
            hip.quantize_mxfp4(W.F32, px, hidden, n, hidden, qc, qs, st)
            up.mul_device(W.MXFP4, qc, qs, hidden, n, off, tok, n * k, W.F32, h, inter, st)
            hip.quantize_mxfp4(W.F32, h, inter, n * k, inter, hc, hs, st)
            down.mul_device(W.MXFP4, hc, hs, inter, n * k, off, 0, n * k, W.F32, y, hidden, st)
        else:
            up.mul_device(W.F32, px, 0, hidden, n, off, tok, n * k, W.F32, h, inter, st)
            down.mul_device(W.F32, h, 0, inter, n * k, off, 0, n * k, W.F32, y, hidden, st)
        hip.combine(W.F32, y, hidden, n * k, pos, wt, n, k, hidden, W.F32, out, hidden, st)

    rt = dev.rt
    st, graph, ex = C.c_void_p(), C.c_void_p(), C.c_void_p()
    try:
        assert rt.hipStreamCreateWithFlags(C.byref(st), 1) == 0
        assert rt.hipStreamBeginCapture(st, 0) == 0
        layer(st.value)
        assert rt.hipStreamEndCapture(st, C.byref(graph)) == 0
        assert rt.hipGraphInstantiate(C.byref(ex), graph, None, None, C.c_size_t(0)) == 0
        for round in range(3):
            x = rng.standard_normal((n, hidden)).astype(f32)
            logits = rng.standard_normal((n, experts)).astype(f32)
            logits[rng.random(logits.shape) < 0.1] = -np.inf
            if n > 1:
                logits[n - 1 - round] = -np.inf  # padding
            dev.fill(px, x)
            dev.fill(pl, logits)
            assert rt.hipGraphLaunch(ex, st) == 0 and rt.hipStreamSynchronize(st) == 0
            got = dev.get(out, (n, hidden)).copy()
            w_ids, w_wt, *_ = _route_expected(logits.astype(np.float64), k, False)
            assert np.array_equal(dev.get(ids, (n, k), i32), w_ids)
            xq = mx_values(*mx_quantize(x.astype(np.float64))) if quantised else x.astype(np.float64)
            want, mag = np.zeros((n, hidden)), np.zeros((n, hidden))
            row_h = dev.get(h, (n * k, inter)).astype(np.float64)
            rows = dev.get(pos, (n, k), i32)
            for t in range(n):
                for j in range(k):
                    e = w_ids[t, j]
                    if e < 0:
                        continue
                    a, ta = _expected(xq[t:t + 1], [g[e], u[e]], True, W.F32, hidden)
                    r = row_h[rows[t, j]]
                    assert np.all(np.abs(r - a[0]) <= ta[0])
                    # from the device's own rows on: quantisation would magnify their rounding
                    hq = mx_values(*mx_quantize(r[None]))[0] if quantised else r
                    want[t] += w_wt[t, j] * (hq @ d[e].T)
                    mag[t] += w_wt[t, j] * (np.abs(hq) @ np.abs(d[e]).T)
            assert np.all(np.abs(got - want) <= (inter + 128 + 64 + k) * 2.0 ** -24 * mag + 1e-44)
            layer(st.value)
            assert rt.hipStreamSynchronize(st) == 0
            assert np.array_equal(dev.get(out, (n, hidden)), got)
    finally:
        for handle, destroy in ((ex, rt.hipGraphExecDestroy), (graph, rt.hipGraphDestroy), (st, rt.hipStreamDestroy)):
            if handle.value:
                destroy(handle)
        up.close()
        down.close()
