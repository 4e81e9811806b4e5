"""Every form of the expert products' kernels and of the routing on the GPU against float64 (the shapes are chosen, and
checked on the CPU, by the library's rules)."""
import numpy as np
import pytest

import expert_forms as F
from experts_fixture import EPS, Device, bits_dtype, decode, encode, matrices, mx_rows, mx_values, random_mx, silu
from test_gpu_experts import _close, _route_expected
from tinyoai_amd import weights as W

pytestmark = pytest.mark.gpu

BASE = 37  # rows of a matrix that differ; the others repeat them


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


def _matrix(rng, fmt, experts, rows, cols):
    """Raw matrices and the float64 values of their first BASE rows."""
    raw, w = matrices(rng, fmt, experts, min(rows, BASE), cols)
    raw = raw.reshape(experts, min(rows, BASE), -1)
    return np.ascontiguousarray(raw[:, np.arange(rows) % BASE]).reshape(-1), w


def _tolerance(x, w, cols):
    """A chain of sums on the matrix cores rounds 512 times at most (8192 columns of planes by 16), each time by 2^-23 of
    the partial sum at most; up to 16 waves' and 4 chains' sums of three planes meet in fp32."""
    return (512 * 2 + 64) * 2.0 ** -24 * (np.abs(x) @ np.abs(w).T)


def _check(got, x, ws, gate, odtype, cols):
    y, t = x @ ws[0].T, _tolerance(x, ws[0], cols)
    if not gate:  # the norm of the error: as of a random walk (a quarter of the root of the roundings, a margin of a half)
        assert np.linalg.norm(got - y) <= (1.5 * 0.25 * np.sqrt(512 + 64) * 2.0 ** -24 + EPS[odtype]) * np.linalg.norm(y)
    if gate:
        u, tu = x @ ws[1].T, _tolerance(x, ws[1], cols)
        s = silu(y)
        t = 1.1 * t * (np.abs(u) + tu) + np.abs(s) * tu + 10 * 2.0 ** -24 * np.abs(s * u)  # |silu'| < 1.1
        y = s * u
    t = t + EPS[odtype] * (np.abs(y) + t) + (2.0 ** -25 if odtype == W.F16 else 1e-44)
    assert np.all(_close(got, y, t, odtype)), np.max(np.abs(got - y) / t)


def _name(c):
    return "-".join(map(str, [*c.form, W.DTYPE_NAMES[c.fmt], W.DTYPE_NAMES[c.xdtype], "pairs" if c.gate else "plain", c.cols]))


@pytest.mark.parametrize("c", [*F.few_forms(), *F.tile_forms()], ids=_name)
def test_product_form(hip, dev, c):
    """Rows picked by an index (two of them name none), wider output rows, rows behind the last group, every output and
    every value that is not one."""
    rng = np.random.default_rng(c.cols + c.rows)
    experts, m = len(c.counts), sum(c.counts)
    n, x_rows, ldo = m + F.TAIL, m // 2 + 2, c.rows + 5
    data = [_matrix(rng, c.fmt, experts, c.rows, c.cols) for _ in range(2 if c.gate else 1)]
    ps, ldx = 0, c.cols
    if c.xdtype == W.MXFP4:
        q = random_mx(rng, x_rows, c.cols, 122, 128)
        x = mx_values(*q)
        px, ps = (dev.put(a) for a in mx_rows(*q))
    else:
        ldx += 8
        bits, x = encode(c.xdtype, rng.standard_normal((x_rows, ldx)))
        px, x = dev.put(bits), x[:, :c.cols]
    index = rng.integers(0, x_rows, n).astype(np.int32)
    index[[0, m - 1]] = [-1, x_rows]
    offsets = np.concatenate([[0], np.cumsum(c.counts)]).astype(np.int32)
    fresh = np.full((n, ldo), 7, bits_dtype(c.odtype))
    e = hip.Experts(c.fmt, experts, c.rows, c.cols, *(d[0] for d in data))
    out = dev.put(fresh)
    e.mul_device(c.xdtype, px, ps, ldx, x_rows, dev.put(offsets), dev.put(index), n, c.odtype, out, ldo)
    raw = dev.get(out, (n, ldo), bits_dtype(c.odtype))
    e.close()
    assert np.array_equal(raw[m:], fresh[m:]) and np.array_equal(raw[:, c.rows:], fresh[:, c.rows:])
    assert not raw[[0, m - 1], :c.rows].any()
    # every repetition of the first rows has their bits
    for r in range(BASE, c.rows, BASE):
        assert np.array_equal(raw[:m, r:min(r + BASE, c.rows)], raw[:m, :min(BASE, c.rows - r)]), r
    first = min(BASE, c.rows)
    got = decode(c.odtype, np.ascontiguousarray(raw[:m, :first]))
    for i in range(experts):
        r = np.arange(max(offsets[i], 1), min(offsets[i + 1], m - 1))
        if r.size:
            _check(got[r], x[index[r]], [d[1][i] for d in data], c.gate, c.odtype, c.cols)


@pytest.mark.parametrize("form,fmt,xdtype,n,rows,cols", [*F.run_forms()])
def test_product_of_runs(hip, dev, form, fmt, xdtype, n, rows, cols):
    """Long rows, whose sums go to totals: no more roundings than fp32 sums of 512 columns have (a run of 1024 columns of
    three planes 192, its totals 64 at most here; MXFP4 rows' of 8192 columns 128 and 17)."""
    rng = np.random.default_rng(cols)
    raw, w = _matrix(rng, fmt, 1, rows, cols)
    at, ps = np.arange(n) % 61, 0
    if xdtype == W.MXFP4:
        q = random_mx(rng, 61, cols, 120, 130)
        x = mx_values(*q)
        px, ps = (dev.put(a) for a in mx_rows(*(a[at] for a in q)))
    else:
        bits, x = encode(xdtype, rng.standard_normal((61, cols)))
        px = dev.put(bits[at])
    out = dev.put(np.full((n, rows), np.nan, np.float32))
    e = hip.Experts(fmt, 1, rows, cols, raw)
    e.mul_device(xdtype, px, ps, cols, n, dev.put(np.array([0, n], np.int32)), 0, n, W.F32, out, rows)
    got = dev.get(out, (n, rows))
    e.close()
    want = x @ w[0].T
    assert np.linalg.norm(got[:61, :BASE] - want) <= 1.5 * 0.25 * np.sqrt(512.0) * 2.0 ** -24 * np.linalg.norm(want)
    assert np.array_equal(got, got[:61, :BASE][at][:, np.arange(rows) % BASE])


@pytest.mark.parametrize("form,n,experts,k", F.ROUTES)
@pytest.mark.parametrize("over_all", [False, True])
def test_routing_form(hip, dev, form, n, experts, k, over_all):
    """Ties, masked experts and tokens; most tokens on a few experts."""
    rng = np.random.default_rng(n * k)
    x = (rng.standard_normal((n, experts)) * 1.5).round(1).astype(np.float32)
    x[:, : max(1, experts // 10)] += 2
    x[rng.random(x.shape) < 0.1] = -np.inf
    x[1], x[2, ::2] = -np.inf, np.nan
    want = _route_expected(x.astype(np.float64), k, over_all)
    shapes = [(n, k), (n, k), (experts + 1,), (n * k,), (n, k)]
    types = [np.int32, np.float32, np.int32, np.int32, np.int32]
    p = [dev.put(np.full(s, 99, t)) for s, t in zip(shapes, types)]
    hip.route(W.F32, dev.put(x), experts, n, experts, k, over_all, *p)
    got = [dev.get(q, s, t) for q, s, t in zip(p, shapes, types)]
    for i in (0, 2, 3, 4):
        assert np.array_equal(got[i], want[i]), i
    # exp, the sum (64 lanes of 16, then 6 steps), the quotient, and the rounding of l - m (2^-24 of 20 in the exponent)
    assert np.all(np.abs(got[1] - want[1]) <= 64 * 2.0 ** -24 * want[1] + 1e-44)
