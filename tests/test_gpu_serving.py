"""Rotary positions, the paged cache, attention over its pages and attention of packed prompts on the GPU against
float64."""
import ctypes as C
import math

import numpy as np
import pytest

from experts_fixture import EPS, Device, bits_dtype, decode, encode
from tinyoai_amd import weights as W

pytestmark = pytest.mark.gpu

TYPES = (W.F32, W.F16, W.BF16)
CACHES = TYPES + (W.Q8_0,)
U = 2.0 ** -24  # half a step of fp32, relative


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


def _rows(rng, dev, dtype, n, width, pad=0, shift=0, spread=1.0):
    """n rows of `width` values of a buffer `pad` wider: (address, distance, float64 values)."""
    bits, x = encode(dtype, rng.standard_normal((n, width + pad)) * spread)
    return dev.put(bits, shift), width + pad, x[:, :width]


def _empty(dev, dtype, n, width, pad=0, shift=0):
    """A buffer whose every value is 7, in bits."""
    return dev.put(np.full((n, width + pad), 7, bits_dtype(dtype)), shift)


def _take(dev, ptr, dtype, n, width, pad=0):
    raw = dev.get(ptr, (n, width + pad), bits_dtype(dtype)).copy()
    assert (raw[:, width:] == 7).all()
    return raw[:, :width]


# ---------------------------------------------------------------- rotary positions
def _angles(positions, hd, rot, theta, scaling="none", factor=1.0, context=0, low=0.0, high=0.0):
    f = theta ** (-2.0 * np.arange(rot // 2) / rot)
    turns = context * f / (2 * np.pi)
    if scaling == "linear":
        f = f / factor
    elif scaling == "bands":
        mix = np.select([turns >= high, turns <= low], [1.0, 0.0], (turns - low) / (high - low))
        f = mix * f + (1 - mix) * f / factor
    elif scaling == "yarn":
        first, last = (rot * math.log(context / (2 * math.pi * t)) / (2 * math.log(theta)) for t in (high, low))
        first, last = max(math.floor(first), 0), min(math.ceil(last), rot - 1)
        mix = np.clip((np.arange(rot // 2) - first) / max(last - first, 0.001), 0, 1)
        f = f * (1 - mix) + f / factor * mix
    return np.asarray(positions, np.float64)[:, None] * f


def _rope_check(hip, dev, rng, n, heads, hd, rot, layout, dtype, odtype, positions, theta=1e4, pad=0, shift=0, **scaling):
    px, ld, x = _rows(rng, dev, dtype, n, heads * hd, pad, shift)
    out = _empty(dev, odtype, n, heads * hd, pad, shift)
    rope = hip.Rope(hd, rot, layout, theta, **scaling)
    rope.rotate(dtype, px, ld, n, heads, dev.put(np.asarray(positions, np.int32)), odtype, out, ld)
    got = decode(odtype, _take(dev, out, odtype, n, heads * hd, pad)).reshape(n, heads, hd)
    rope.close()
    a = _angles(positions, hd, rot, theta, **scaling)[:, None]
    m = 0.1 * math.log(scaling["factor"]) + 1 if scaling.get("scaling") == "yarn" else 1.0
    x = x.reshape(n, heads, hd)
    i, j = (np.arange(rot // 2), np.arange(rot // 2) + rot // 2) if layout == "half" else (np.arange(0, rot, 2), np.arange(1, rot, 2))
    want, mag = x.copy(), np.zeros_like(x)
    want[..., i], want[..., j] = m * (x[..., i] * np.cos(a) - x[..., j] * np.sin(a)), m * (x[..., j] * np.cos(a) + x[..., i] * np.sin(a))
    mag[..., i] = mag[..., j] = np.abs(x[..., i]) + np.abs(x[..., j])
    # the angle in [-pi, pi] is rounded to fp32 (2^-23 at most), sine and cosine are off by two units at most (2^-23),
    # their product with m, the two products and the sum round once each; the result rounds to its type
    tol = mag * m * (2.0 ** -23 + 2.0 ** -23 + 4 * U) + EPS[odtype] * np.abs(want) + (2.0 ** -25 if odtype == W.F16 else 0)
    assert np.all(np.abs(got - want) <= tol)
    if dtype == odtype:
        assert np.array_equal(got[..., rot:], x[..., rot:])


@pytest.mark.parametrize("dtype,odtype", [(W.F32, W.F32), (W.F16, W.F16), (W.BF16, W.BF16), (W.F32, W.BF16), (W.BF16, W.F32)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope(hip, dev, dtype, odtype, layout):
    rng = np.random.default_rng(1)
    for n, heads, hd, rot, pad, shift in ((1, 1, 8, 2, 0, 0), (5, 64, 80, 20, 0, 0), (3, 7, 64, 64, 1, 4), (33, 12, 128, 128, 8, 0),
                                          (2, 3, 256, 250, 3, 8), (70, 2, 72, 36, 0, 4)):
        positions = rng.integers(0, 100000, n)
        _rope_check(hip, dev, rng, n, heads, hd, rot, layout, dtype, odtype, positions, pad=pad, shift=shift)


@pytest.mark.parametrize("scaling", [dict(scaling="linear", factor=4.0), dict(scaling="bands", factor=8.0, context=8192, low=1.0, high=4.0),
                                     dict(scaling="yarn", factor=16.0, context=4096, low=1.0, high=32.0)])
def test_rope_scalings(hip, dev, scaling):
    rng = np.random.default_rng(2)
    for rot, theta in ((128, 5e5), (64, 1e4), (10, 1e4)):
        positions = np.concatenate([[0, 1, -5, 131071, 1 << 20], rng.integers(0, 40000, 20)])
        _rope_check(hip, dev, rng, 25, 4, 128, rot, "half", W.F32, W.F32, positions, theta, **scaling)


def test_rope_far_positions_and_in_place(hip, dev):
    """Positions up to 2^30, whose float64 angles are off by 2^-23 rad themselves; rows turned in place."""
    rng = np.random.default_rng(3)
    positions = np.array([1 << 24, (1 << 24) + 1, 1 << 26, -(1 << 26)])
    _rope_check(hip, dev, rng, 4, 3, 64, 64, "half", W.F32, W.F32, positions)
    for layout in ("half", "interleaved"):
        for dtype in TYPES:
            for hd, rot in ((80, 20), (64, 64), (72, 30)):
                px, ld, _ = _rows(rng, dev, dtype, 9, 5 * hd, 3)
                raw = dev.get(px, (9, ld), bits_dtype(dtype)).copy()
                out, pp = dev.put(raw), dev.put(np.arange(9, dtype=np.int32) * 100)
                rope = hip.Rope(hd, rot, layout)
                rope.rotate(dtype, px, ld, 9, 5, pp, dtype, out, ld)
                rope.rotate(dtype, px, ld, 9, 5, pp, dtype, px, ld)
                rope.close()
                got = dev.get(px, (9, ld), bits_dtype(dtype))
                assert np.array_equal(got, dev.get(out, (9, ld), bits_dtype(dtype)))
                assert np.array_equal(got[:, 5 * hd:], raw[:, 5 * hd:]) and not np.array_equal(got, raw)
    with pytest.raises(hip.TinyoaiError, match="in place"):
        r = hip.Rope(64, 64)
        r.rotate(W.F32, px, 512, 1, 1, pp, W.F16, px, 512)


# ---------------------------------------------------------------- the paged cache
def _held(dtype, x, hd):
    """What a cache of this type stands for, of float64 rows [n, heads * hd] that fp32 holds."""
    if dtype != W.Q8_0:
        with np.errstate(over="ignore"):
            return encode(dtype, x)[1] if dtype != W.BF16 else _bf16(x)
    b = x.reshape(*x.shape[:-1], -1, hd)
    out = np.empty_like(b)
    for c in range(0, hd, 32):
        v = b[..., c:c + 32].astype(np.float32)
        finite = np.isfinite(v).all(-1, keepdims=True)
        v = np.where(finite, v, 0)
        most = np.abs(v).max(-1, keepdims=True)
        with np.errstate(over="ignore"):
            d = np.minimum(most / np.float32(127), np.float32(65504)).astype(np.float16).astype(np.float32)
        q = np.clip(np.rint(v / np.where(d > 0, d, np.float32(1))), -127, 127)
        q = np.where(d > 0, q, 0).astype(np.float64)
        out[..., c:c + 32] = np.where(finite, q * d.astype(np.float64), np.nan)
    return out.reshape(x.shape)


def _bf16(x):
    x = np.asarray(x, np.float32)
    return np.where(np.isfinite(x), encode(W.BF16, np.where(np.isfinite(x), x, 0))[1], x.astype(np.float64))


def _edges(rng, n, width):
    """Rows with blocks of zeros, tiny and huge values, halfway codes and values that are not finite."""
    x = (rng.standard_normal((n, width)) * np.exp(rng.standard_normal(width))).astype(np.float32)
    if n >= 8 and width >= 32:
        x[0, :32] = 0
        x[1, :32] *= np.float32(1e-9)
        x[2, :32] *= np.float32(1e30)
        x[3, :8] = [127, .5, 1.5, -2.5, 126.5, -126.5, 63.5, 0]
        x[4, 3], x[5, 4], x[6, 5] = np.inf, np.nan, -np.inf
        x[7, :8] = [1e-7, -3e-7, 5e-8, 0, -0.0, 2e-7, 1e-6, 3e-6]
    return x


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cache", CACHES)
def test_cache_rows(hip, dev, cache, dtype):
    """Written rows read back as the values that the cache's type holds, bit for bit; rows of slots outside the cache are
    left out and read as zeros; other slots and layers keep what they hold."""
    rng = np.random.default_rng(4)
    for n, heads, hd, page, pad, shift in ((1, 1, 8, 1, 0, 0), (9, 3, 72, 4, 1, 4), (40, 8, 128, 16, 0, 0), (300, 2, 80, 64, 5, 8),
                                           (11, 2, 256, 1024, 0, 4), (20, 3, 40, 8, 2, 0)):
        width, pages = heads * hd, -(-(n + 9) // page) + 1
        c = hip.KVPages(cache, 2, heads, hd, page, pages)
        with np.errstate(over="ignore", invalid="ignore"):
            (kb, k), (vb, v) = (_encoded(dtype, _edges(rng, n, width + pad)) for _ in range(2))
        pk, pv = dev.put(kb, shift), dev.put(vb, shift)
        slots = rng.permutation(pages * page)[:n].astype(np.int32)
        ok = np.ones(n, bool)
        if n > 8:
            slots[[2, 5, 8]] = [-1, pages * page, -(1 << 31)]
            ok[[2, 5, 8]] = False
        ps = dev.put(slots)
        c.write(1, dtype, pk, width + pad, pv, width + pad, ps, n)
        for odtype in TYPES:
            ko, vo = _empty(dev, odtype, n, width, pad, shift), _empty(dev, odtype, n, width, pad, shift)
            c.read(1, odtype, ko, width + pad, vo, width + pad, ps, n)
            for out, x in ((ko, k), (vo, v)):
                with np.errstate(over="ignore", invalid="ignore"):
                    want = _held(cache, x[:, :width], hd)
                    want = np.where(ok[:, None], want, 0)
                    want = _encoded(odtype, want)[1]
                got = decode(odtype, _take(dev, out, odtype, n, width, pad))
                assert np.array_equal(got, want, equal_nan=True)
        # every other slot, and the other layer, still holds zeros
        rest = np.setdiff1d(np.arange(pages * page), slots).astype(np.int32)
        for layer, s in ((1, rest), (0, np.arange(pages * page, dtype=np.int32))):
            ko, vo = _empty(dev, W.F32, len(s), width), _empty(dev, W.F32, len(s), width)
            c.read(layer, W.F32, ko, width, vo, width, dev.put(s), len(s))
            assert not dev.get(ko, (len(s), width)).any() and not dev.get(vo, (len(s), width)).any()
        c.close()


def _encoded(dtype, x):
    """encode() of values that may not be finite."""
    x = np.asarray(x, np.float32)
    if dtype != W.BF16:
        return encode(dtype, x)
    v = _bf16(x).astype(np.float32)
    return (v.view(np.uint32) >> 16).astype(np.uint16), v.astype(np.float64)


# ---------------------------------------------------------------- attention
def _attention(q, k, v, scale, seen=None):
    """(outputs, sums of weight times magnitude, the largest sums of scale |q| |k|) of queries [m, hd] in float64; a query
    without keys gets zeros."""
    out, mag, load = np.zeros((len(q), v.shape[1])), np.zeros((len(q), v.shape[1])), np.zeros((len(q), 1))
    if not len(k):
        return out, mag, load
    s = q @ k.T * scale
    a = np.abs(q) @ np.abs(k).T * scale
    if seen is not None:
        s, a = np.where(seen, s, -np.inf), np.where(seen, a, 0)
    top = s.max(-1, keepdims=True)
    p = np.exp(s - np.where(np.isfinite(top), top, 0))
    total = p.sum(-1, keepdims=True)
    p = np.where(total > 0, p / np.where(total > 0, total, 1), 0)
    return p @ v, p @ np.abs(v), a.max(-1, keepdims=True)


def _tolerance(want, mag, load, keys, hd, dtype, rounded):
    """Scores are sums of hd products and two products more, each rounded (U of the sums of magnitudes), so weights are off
    by twice that, by the power's and the subtraction's roundings (8 U, and the score's magnitude times 2 U) and, where they
    are rounded to a type, by half a step of that (`rounded`); sums of `keys` terms, spread over at least four chains, then
    joined, round that often. The result rounds to its type; weights that fall below 2^-126 or a type's range vanish."""
    weight = 2 * (hd + 4) * U * load + 8 * U + rounded
    chain = (keys / 4 + 64) * U
    return mag * (2 * weight + 2 * chain) * 1.01 + EPS[dtype] * np.abs(want) + keys * 2.0 ** -100 + (2.0 ** -24 if dtype == W.F16 else 0)


def _attend_check(hip, dev, rng, cache, dtype, heads, kv, hd, page, lengths, pad=0, shift=0, drop=0.0, spread=1.0, poison=True):
    """New tokens of sequences of these lengths over pages in any order. Every value behind a sequence's last position, and
    every page that no table names, is NaN; table entries past the length name no page."""
    n, width = len(lengths), max(1, -(-max(max(lengths), 1) // page))
    used = sum(-(-max(x, 0) // page) for x in lengths)
    pages = used + 3
    order = rng.permutation(pages)[:used]
    table = np.full((n, width), -7, np.int32)
    at = 0
    for i, x in enumerate(lengths):
        m = -(-max(x, 0) // page)
        table[i, :m] = order[at:at + m]
        at += m
    gone = (rng.random(table.shape) < drop) & (table >= 0)
    bad = table.copy()
    bad[gone] = rng.choice([-1, pages, 1 << 30], gone.sum())
    kvw, qw = kv * hd, heads * hd
    (kx, vx) = (rng.standard_normal((pages * page, kvw)).astype(np.float32) * np.float32(spread) for _ in range(2))
    live = np.zeros(pages * page, bool)
    for i, x in enumerate(lengths):
        t = np.arange(max(x, 0))
        live[table[i, t // page] * page + t % page] = True
    if poison:
        kx[~live] = vx[~live] = np.nan
    c = hip.KVPages(cache, 1, kv, hd, page, pages)
    c.write(0, W.F32, dev.put(kx), kvw, dev.put(vx), kvw, dev.put(np.arange(pages * page, dtype=np.int32)), pages * page)
    pq, ldq, q = _rows(rng, dev, dtype, n, qw, pad, shift)
    out = _empty(dev, dtype, n, qw, pad, shift)
    scale = hd ** -0.5
    c.attend(0, dtype, pq, ldq, heads, scale, dev.put(bad), width, dev.put(np.asarray(lengths, np.int32)), n, out, ldq)
    got = decode(dtype, _take(dev, out, dtype, n, qw, pad)).reshape(n, heads, hd)
    with np.errstate(invalid="ignore"):
        k, v = (_held(cache, x.astype(np.float64), hd).reshape(-1, kv, hd) for x in (kx, vx))
    for i, x in enumerate(lengths):
        t = np.arange(max(x, 0))
        t = t[~gone[i, t // page]]
        slots = table[i, t // page] * page + t % page
        for h in range(heads):
            g = h // (heads // kv)
            want, mag, load = _attention(q[i].reshape(heads, hd)[h:h + 1], k[slots, g], v[slots, g], scale)
            tol = _tolerance(want, mag, load, len(t), hd, dtype, _weights_rounded(cache, dtype))
            assert np.all(np.abs(got[i, h] - want[0]) <= tol[0]), (i, h, x)
            if not len(t):
                assert not got[i, h].any()
    c.close()


def _weights_rounded(cache, dtype):
    """New tokens' weights: fp32 in all their bits, or for 16-bit results two planes of eight bits, the second cut short
    (what a plane leaves is below 2^-7 of what it was)."""
    return 0.0 if dtype == W.F32 or cache == W.F32 else 2.0 ** -14


ATTEND = [(1, 1, 8, 1, (1,)), (8, 4, 8, 16, (1, 0, 5, 160)), (4, 4, 80, 64, (700, 1, 63, 64, 65)), (8, 2, 64, 16, (17, 0, 300, 15)),
          (6, 2, 72, 32, (130, 31, 33)), (16, 1, 128, 128, (129, 257, 1)), (12, 4, 256, 8, (40, 9, 8)), (5, 1, 96, 4, (3, 100)),
          (20, 1, 64, 64, (90, 64)), (34, 2, 40, 16, (50,)), (3, 1, 160, 16, (70, 33)), (2, 2, 200, 32, (64,))]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cache", CACHES)
def test_attend(hip, dev, cache, dtype):
    rng = np.random.default_rng(5)
    for heads, kv, hd, page, lengths in ATTEND:
        _attend_check(hip, dev, rng, cache, dtype, heads, kv, hd, page, lengths)


@pytest.mark.parametrize("cache", CACHES)
def test_attend_long(hip, dev, cache):
    """Sequences over several blocks, ranges that end anywhere, entries that name no page, odd strides and alignments."""
    rng = np.random.default_rng(6)
    dtype = W.F16 if cache == W.F16 else W.F32
    _attend_check(hip, dev, rng, cache, dtype, 8, 2, 64, 16, (5000, 2049, 0, 511, 513), pad=3, shift=4)
    _attend_check(hip, dev, rng, cache, dtype, 2, 2, 128, 256, (9000, 1), drop=0.2)
    _attend_check(hip, dev, rng, cache, W.BF16, 3, 1, 80, 8, (4097, 20, 300), pad=1, shift=2, drop=0.5)
    _attend_check(hip, dev, rng, cache, dtype, 16, 2, 128, 64, tuple(rng.integers(0, 900, 40)))
    _attend_check(hip, dev, rng, cache, dtype, 2, 1, 8, 4, tuple(rng.integers(0, 3, 200)) + (600, 0, 129) + (1,) * 70)
    _attend_check(hip, dev, rng, cache, dtype, 3, 3, 64, 32, tuple(rng.integers(0, 300, 130)))


@pytest.mark.parametrize("cache", CACHES)
def test_attend_large_scores(hip, dev, cache):
    """Scores of hundreds: a softmax that is all on one position, wherever it lies."""
    rng = np.random.default_rng(7)
    _attend_check(hip, dev, rng, cache, W.F32, 4, 1, 128, 16, (1500, 40), spread=20.0)
    _attend_check(hip, dev, rng, cache, W.F32, 2, 2, 64, 16, (1500, 40), spread=1e-3)


def test_attend_entries(hip, dev):
    """All entries outside the pool, lengths beyond the table, negative lengths: zeros or the table's positions."""
    rng = np.random.default_rng(8)
    hd, page, pages = 64, 16, 4
    c = hip.KVPages(W.F16, 1, 1, hd, page, pages)
    bits, kv = encode(W.F16, rng.standard_normal((pages * page, hd)))
    p = dev.put(bits)
    c.write(0, W.F16, p, hd, p, hd, dev.put(np.arange(64, dtype=np.int32)), 64)
    table = np.array([[0, 1], [-1, 4], [2, 3], [1 << 30, -(1 << 31)], [3, 0]], np.int32)
    lengths = np.array([1000, 32, -5, 20, 2**31 - 1], np.int32)
    pq, _, q = _rows(rng, dev, W.F32, 5, hd)
    out = _empty(dev, W.F32, 5, hd)
    c.attend(0, W.F32, pq, hd, 1, 0.125, dev.put(table), 2, dev.put(lengths), 5, out, hd)
    got = dev.get(out, (5, hd)).astype(np.float64)
    for i, slots in ((0, np.arange(32)), (4, np.concatenate([np.arange(48, 64), np.arange(16)]))):
        want, mag, load = _attention(q[i:i + 1], kv[slots], kv[slots], 0.125)
        assert np.all(np.abs(got[i] - want[0]) <= _tolerance(want, mag, load, 32, hd, W.F32, 0)[0])
    assert not got[1:4].any()
    for bad in (dict(heads=0), dict(width=0), dict(n=-1), dict(table=None), dict(lengths=None), dict(scale=math.nan), dict(layer=1),
                dict(layer=-1), dict(width=1 << 28), dict(n=1 << 30), dict(q=None), dict(ldq=63)):
        a = dict(layer=0, q=pq, ldq=hd, heads=1, scale=1.0, table=p, width=2, lengths=p, n=1) | bad
        with pytest.raises(hip.TinyoaiError):
            c.attend(a["layer"], W.F32, a["q"], a["ldq"], a["heads"], a["scale"], a["table"], a["width"], a["lengths"], a["n"], out, hd)
    two = hip.KVPages(W.F16, 1, 2, hd, page, 1)
    with pytest.raises(hip.TinyoaiError, match="query heads"):
        two.attend(0, W.F32, pq, 3 * hd, 3, 1.0, p, 1, p, 1, out, 3 * hd)
    two.close()
    c.attend(0, W.F32, pq, hd, 1, 1.0, p, 1, p, 0, out, hd)
    c.close()


def test_attend_full_tables(hip, dev):
    """64 sequences that each fill the longest table (its entries all one page): 2^31 units of 32 positions, one
    more than 31 bits count. Equal scores and small whole values, so that every sum is exact: multiples of 32
    up to 2^30 times at most 8."""
    hd, page, width, n = 8, 1024, 1 << 20, 64
    c = hip.KVPages(W.BF16, 1, 1, hd, page, 1)
    k, v = encode(W.BF16, np.zeros((page, hd)))[0], encode(W.BF16, np.tile(np.arange(1.0, 9.0), (page, 1)))[0]
    c.write(0, W.BF16, dev.put(k), hd, dev.put(v), hd, dev.put(np.arange(page, dtype=np.int32)), page)
    out = _empty(dev, W.F32, n, hd)
    c.attend(0, W.F32, dev.put(np.ones((n, hd), np.float32)), hd, 1, 1.0, dev.put(np.zeros((n, width), np.int32)), width,
             dev.put(np.full(n, 2**31 - 1, np.int32)), n, out, hd)
    assert np.array_equal(dev.get(out, (n, hd)), np.tile(np.arange(1.0, 9.0, dtype=np.float32), (n, 1)))
    c.close()


# ---------------------------------------------------------------- packed prompts
def _prompt_check(hip, dev, rng, dtype, heads, kv, hd, lengths, causal, pad=0, shift=0, spread=1.0, hidden=False):
    """Sequences of (queries, keys); two rows more than theirs in every buffer. `hidden`: values that are not finite in keys
    and values that only some queries see."""
    nq, nk = (sum(x[i] for x in lengths) + 2 for i in range(2))
    (pq, ldq, q), (pk, ldk, k), (pv, ldv, v) = (_rows(rng, dev, dtype, m, h * hd, pad, shift, spread) for m, h in ((nq, heads), (nk, kv), (nk, kv)))
    if hidden:
        for p, x in ((pk, k), (pv, v)):
            raw = dev.get(p, (nk, kv * hd + pad), bits_dtype(dtype)).copy()
            x[-2:] = np.nan
            at = 0
            for m, keys in lengths:
                if keys > 3:
                    x[at + keys - 1, ::3] = np.nan
                    x[at + keys - 2, 1::3] = np.inf
                    x[at + keys // 2, 2::7] = -np.inf
                at += keys
            raw[:, :kv * hd] = _encoded(dtype, x)[0]
            dev.fill(p, raw)
    qo, ko = (np.cumsum([0] + [x[i] for x in lengths]).astype(np.int32) for i in range(2))
    out = _empty(dev, dtype, nq, heads * hd, pad, shift)
    scale = hd ** -0.5
    hip.attention(dtype, pq, ldq, heads, pk, ldk, pv, ldv, kv, hd, scale, causal, dev.put(qo), dev.put(ko), len(lengths), nq, nk, out, ldq)
    raw = _take(dev, out, dtype, nq, heads * hd, pad)
    assert (raw[-2:] == 7).all()
    got = decode(dtype, raw).reshape(nq, heads, hd)
    for (m, keys), q0, k0 in zip(lengths, qo, ko):
        seen = np.arange(keys) <= np.arange(m)[:, None] + keys - m if causal else None
        for h in range(heads):
            g = slice(h // (heads // kv) * hd, h // (heads // kv) * hd + hd)
            qs, ks, vs = q[q0:q0 + m, h * hd:h * hd + hd], k[k0:k0 + keys, g], v[k0:k0 + keys, g]
            if not hidden:
                want, mag, load = _attention(qs, ks, vs, scale, seen)
                fine = np.ones(want.shape, bool)
            else:  # what a query sees that is not finite makes its outputs so: those of values, column by column
                bad_k, bad_v = ~np.isfinite(ks).all(-1), ~np.isfinite(vs)
                want, mag, load = _attention(qs, np.where(np.isfinite(ks), ks, 0), np.where(bad_v, 0, vs), scale, seen)
                fine = ~((seen @ bad_k.astype(float))[:, None] + seen @ bad_v.astype(float) > 0)
                with np.errstate(invalid="ignore"):  # (a score of -inf is a weight of zero: such a key need not show)
                    zero = (seen & (qs @ ks.T == -np.inf)).any(-1)
                assert not np.isfinite(got[q0:q0 + m, h][~fine & ~zero[:, None]]).any()
            tol = _tolerance(want, mag, load, keys, hd, dtype, 0 if dtype == W.F32 else EPS[dtype])
            assert np.all((np.abs(got[q0:q0 + m, h] - want) <= tol) | ~fine), (m, keys, h)
            if causal and m > keys:
                assert not got[q0:q0 + m - keys, h].any()


PROMPTS = [(1, 1, 8, ((1, 1),)), (8, 4, 8, ((5, 5), (0, 0), (64, 64), (1, 1))), (4, 4, 80, ((19, 449), (130, 130))),
           (8, 2, 64, ((33, 33), (200, 77), (7, 0), (129, 300))), (4, 1, 72, ((65, 65), (3, 190))), (16, 2, 128, ((150, 150), (1, 257))),
           (2, 1, 256, ((70, 131), (128, 128))), (3, 3, 96, ((31, 32), (140, 63))), (6, 2, 40, ((90, 90),)), (1, 1, 160, ((50, 99),)), (2, 1, 200, ((33, 40),))]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
def test_prompt(hip, dev, dtype, causal):
    rng = np.random.default_rng(9)
    for heads, kv, hd, lengths in PROMPTS:
        _prompt_check(hip, dev, rng, dtype, heads, kv, hd, lengths, causal)


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_strides(hip, dev, dtype):
    """Wider rows at odd distances and alignments; many short sequences; scores of hundreds."""
    rng = np.random.default_rng(10)
    for pad, shift in ((1, 4), (3, 2 if dtype != W.F32 else 8), (8, 0), (64, 0)):
        _prompt_check(hip, dev, rng, dtype, 4, 2, 64, ((70, 70), (40, 150)), True, pad, shift)
        _prompt_check(hip, dev, rng, dtype, 2, 2, 128, ((140, 140),), False, pad, shift)
    _prompt_check(hip, dev, rng, dtype, 2, 1, 64, tuple((int(x), int(x)) for x in rng.integers(0, 5, 150)), True)
    _prompt_check(hip, dev, rng, dtype, 2, 1, 128, ((100, 400),), True, spread=5.0)
    _prompt_check(hip, dev, rng, dtype, 1, 1, 80, ((700, 700), (20, 1300)), True)


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_parts(hip, dev, dtype):
    """Few queries over many keys: tiles whose keys are cut into parts, some of them past a short sequence's end."""
    rng = np.random.default_rng(16)
    for heads, kv, hd, lengths in ((4, 2, 64, ((130, 4500),)), (3, 1, 80, ((40, 2100), (200, 4300))), (2, 1, 128, ((1, 7000),)),
                                   (8, 1, 128, ((33, 90), (128, 9000))), (2, 2, 256, ((70, 3000),)), (1, 1, 8, ((300, 6000), (9, 4)))):
        for causal in (True, False):
            _prompt_check(hip, dev, rng, dtype, heads, kv, hd, lengths, causal)
    _prompt_check(hip, dev, rng, dtype, 2, 1, 64, ((150, 4500), (130, 90)), True, hidden=True)
    _prompt_check(hip, dev, rng, dtype, 2, 1, 80, ((20, 400), (5, 5)), True, hidden=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_hidden_values(hip, dev, dtype):
    """Infinities and NaN in keys and values: queries that do not see them are not touched by them."""
    rng = np.random.default_rng(11)
    for hd in (64, 80, 128, 256):
        _prompt_check(hip, dev, rng, dtype, 2, 1, hd, ((5, 5), (64, 64), (90, 130), (200, 200), (17, 5)), True, hidden=True)


def test_prompt_offsets(hip, dev):
    """Offsets that leave the buffers count as the nearest that do not; rows of no sequence stay as they are."""
    rng = np.random.default_rng(12)
    for dtype in TYPES:
        pq, ld, q = _rows(rng, dev, dtype, 20, 64)
        out = _empty(dev, dtype, 20, 64)
        qo, ko = (dev.put(np.array(x, np.int32)) for x in ([-3, 5, 5, 9, 1 << 30], [-100, 4, 8, 8, 2**31 - 1]))
        hip.attention(dtype, pq, 64, 1, pq, 64, pq, 64, 1, 64, 0.125, False, qo, ko, 4, 18, 20, out, 64)
        raw = dev.get(out, (20, 64), bits_dtype(dtype)).copy()
        assert (raw[18:] == 7).all()
        got = decode(dtype, raw)
        for q0, q1, k0, k1 in ((0, 5, 0, 4), (5, 9, 8, 8), (9, 18, 8, 20)):
            want, mag, load = _attention(q[q0:q1], q[k0:k1], q[k0:k1], 0.125)
            assert np.all(np.abs(got[q0:q1] - want) <= _tolerance(want, mag, load, 20, 64, dtype, 0 if dtype == W.F32 else EPS[dtype]))


@pytest.mark.parametrize("scale", [-0.3, 0.0, 7.0])
def test_scales(hip, dev, scale):
    """Scales of any sign, and zero: the mean of the values."""
    rng = np.random.default_rng(18)
    for dtype in TYPES:
        hd, n, keys = 64, 40, 70
        (pq, _, q), (pk, _, k), (pv, _, v) = (_rows(rng, dev, dtype, m, hd) for m in (n, keys, keys))
        out = _empty(dev, dtype, n, hd)
        hip.attention(dtype, pq, hd, 1, pk, hd, pv, hd, 1, hd, scale, False, dev.put(np.array([0, n], np.int32)),
                      dev.put(np.array([0, keys], np.int32)), 1, n, keys, out, hd)
        s = q @ k.T * scale
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        want, mag, load = p @ v, p @ np.abs(v), (np.abs(q) @ np.abs(k).T * abs(scale)).max(-1, keepdims=True)
        tol = _tolerance(want, mag, load, keys, hd, dtype, 0 if dtype == W.F32 else EPS[dtype])
        assert np.all(np.abs(decode(dtype, dev.get(out, (n, hd), bits_dtype(dtype))) - want) <= tol)
        for cache in CACHES:
            c = hip.KVPages(cache, 1, 1, hd, 16, 5)
            c.write(0, dtype, pk, hd, pv, hd, dev.put(np.arange(keys, dtype=np.int32)), keys)
            c.attend(0, dtype, pq, hd, 1, scale, dev.put(np.tile(np.arange(5, dtype=np.int32), n)), 5,
                     dev.put(np.full(n, keys, np.int32)), n, out, hd)
            kc, vc = _held(cache, k, hd), _held(cache, v, hd)
            s = q @ kc.T * scale
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            want, mag, load = p @ vc, p @ np.abs(vc), (np.abs(q) @ np.abs(kc).T * abs(scale)).max(-1, keepdims=True)
            tol = _tolerance(want, mag, load, keys, hd, dtype, _weights_rounded(cache, dtype))
            assert np.all(np.abs(decode(dtype, dev.get(out, (n, hd), bits_dtype(dtype))) - want) <= tol), cache
            c.close()


@pytest.mark.parametrize("cache,page", [(W.F32, 1024), (W.F16, 8)])
def test_pool_past_32_bits(hip, dev, cache, page):
    """A pool whose planes pass 4 GiB: rows at both ends."""
    rng = np.random.default_rng(19)
    heads, hd = 8, 256
    pages = (5 << 30) // (page * heads * hd * (4 if cache == W.F32 else 2))
    c = hip.KVPages(cache, 1, heads, hd, page, pages)
    table = np.array([[pages - 1, 0, pages - 2]], np.int32)
    length = 2 * page + 5
    t = np.arange(length)
    slots = (table[0, t // page] * page + t % page).astype(np.int32)
    (pk, ld, k), (pv, _, v), (pq, _, q) = (_rows(rng, dev, W.F32, n, heads * hd) for n in (length, length, 1))
    ps = dev.put(slots)
    c.write(0, W.F32, pk, ld, pv, ld, ps, length)
    ko, vo, out = (_empty(dev, W.F32, n, heads * hd) for n in (length, length, 1))
    c.read(0, W.F32, ko, ld, vo, ld, ps, length)
    k, v = _held(cache, k, hd), _held(cache, v, hd)
    assert np.array_equal(dev.get(ko, k.shape), k) and np.array_equal(dev.get(vo, v.shape), v)
    c.attend(0, W.F32, pq, ld, heads, 0.0625, dev.put(table), 3, dev.put(np.array([length], np.int32)), 1, out, ld)
    got = dev.get(out, (heads, hd))
    for h in range(heads):
        g = slice(h * hd, h * hd + hd)
        want, mag, load = _attention(q[:, g], k[:, g], v[:, g], 0.0625)
        assert np.all(np.abs(got[h] - want[0]) <= _tolerance(want, mag, load, length, hd, W.F32, 0)[0])
    c.close()


def test_prompt_past_32_bits(hip, dev):
    """Rows of keys and values 8 MiB apart, 5.6 GiB of them."""
    rng = np.random.default_rng(20)
    hd, n, keys, ld = 64, 50, 700, 1 << 22
    buf = dev.room((keys * ld + 2 * hd) * 2)
    (kb, k), (vb, v) = (encode(W.F16, rng.standard_normal((keys, hd))) for _ in range(2))
    both = np.concatenate([kb, vb], 1)
    for r in range(keys):
        row = np.ascontiguousarray(both[r])
        assert dev.rt.hipMemcpy(buf + r * ld * 2, row.ctypes.data, row.nbytes, 1) == 0
    pq, _, q = _rows(rng, dev, W.F16, n, hd)
    out = _empty(dev, W.F16, n, hd)
    hip.attention(W.F16, pq, hd, 1, buf, ld, buf + 2 * hd, ld, 1, hd, 0.125, True, dev.put(np.array([0, n], np.int32)),
                  dev.put(np.array([0, keys], np.int32)), 1, n, keys, out, hd)
    seen = np.arange(keys) <= np.arange(n)[:, None] + keys - n
    want, mag, load = _attention(q, k, v, 0.125, seen)
    tol = _tolerance(want, mag, load, keys, hd, W.F16, EPS[W.F16])
    assert np.all(np.abs(decode(W.F16, dev.get(out, (n, hd), np.uint16)) - want) <= tol)


# ---------------------------------------------------------------- streams, graphs, threads
def test_captured_and_concurrent_attention(hip, dev):
    """Two graphs of one cache's long attention and eager calls on a third stream, all in flight together, give an eager
    call's bits on every replay, with eager work between the replays."""
    rng = np.random.default_rng(13)
    heads, kv, hd, page, n, length, rt = 8, 2, 64, 16, 3, 6000, dev.rt
    width = -(-length // page)
    c = hip.KVPages(W.BF16, 1, kv, hd, page, n * width)
    rows = n * width * page
    pk, ld, _ = _rows(rng, dev, W.BF16, rows, kv * hd)
    c.write(0, W.BF16, pk, ld, pk, ld, dev.put(np.arange(rows, dtype=np.int32)), rows)
    table = dev.put(rng.permutation(n * width).astype(np.int32))
    lengths = [dev.put(np.array(x, np.int32)) for x in ([6000, 10, 3000], [0, 6000, 5999], [6000, 6000, 6000])]
    qs = [_rows(rng, dev, W.F32, n, heads * hd)[0] for _ in range(3)]
    y = [dev.put(np.zeros((n, heads * hd), np.float32)) for _ in range(4)]
    streams, execs = [C.c_void_p() for _ in range(3)], []

    def call(i, out, stream=0):
        c.attend(0, W.F32, qs[i], heads * hd, heads, 0.125, table, width, lengths[i], n, out, heads * hd, stream)

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
            want.append(dev.get(y[3], (n, heads * hd)).copy())
        assert all(np.abs(x).max() > 0 for x in want)
        for _ in range(3):
            for i in range(3):
                dev.fill(y[i], np.zeros((n, heads * hd), np.float32))
            for _ in range(4):
                for i in range(2):
                    assert rt.hipGraphLaunch(execs[i], streams[i]) == 0
                call(2, y[2], streams[2].value)
            for i in range(3):
                assert np.array_equal(dev.get(y[i], (n, heads * hd)), want[i]), i
    finally:
        for ex in execs:
            rt.hipGraphExecDestroy(ex)
        for st in streams:
            rt.hipStreamDestroy(st)
        c.close()


@pytest.mark.parametrize("dtype,n,keys", [(W.F32, 19, 449), (W.BF16, 130, 6000)])
def test_captured_and_concurrent_prompts(hip, dev, dtype, n, keys):
    """Prompts whose keys are cut into parts: two graphs captured on two streams and eager calls on a third, all in flight
    together, with eager work between the replays."""
    rng = np.random.default_rng(17)
    heads, hd, rt = 4, 64, dev.rt
    qo, ko = dev.put(np.array([0, n], np.int32)), dev.put(np.array([0, keys], np.int32))
    xs = [[_rows(rng, dev, dtype, m, heads * hd)[0] for m in (n, keys, keys)] for _ in range(3)]
    bits = bits_dtype(dtype)
    y = [dev.put(np.zeros((n, heads * hd), bits)) for _ in range(4)]
    streams, execs = [C.c_void_p() for _ in range(3)], []

    def call(i, out, stream=0):
        q, k, v = xs[i]
        hip.attention(dtype, q, heads * hd, heads, k, heads * hd, v, heads * hd, heads, hd, 0.125, True, qo, ko, 1, n, keys, out,
                      heads * hd, stream)

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
            want.append(dev.get(y[3], (n, heads * hd), bits).copy())
        assert all(x.any() for x in want)
        for _ in range(3):
            for i in range(3):
                dev.fill(y[i], np.zeros((n, heads * hd), bits))
            for _ in range(4):
                for i in range(2):
                    assert rt.hipGraphLaunch(execs[i], streams[i]) == 0
                call(2, y[2], streams[2].value)
            for i in range(3):
                assert np.array_equal(dev.get(y[i], (n, heads * hd), bits), want[i]), i
    finally:
        for ex in execs:
            rt.hipGraphExecDestroy(ex)
        for st in streams:
            rt.hipStreamDestroy(st)


@pytest.mark.parametrize("cache,dtype", [(W.F16, W.F32), (W.Q8_0, W.F32), (W.BF16, W.BF16), (W.F32, W.F32)])
def test_serving_layer(hip, dev, cache, dtype):
    """A layer's attention as a server runs it, one stream: two prompts' rotated rows through the packed attention and into
    pages, a second chunk of one of them over what is read back, then decode steps from one captured graph whose buffers are
    refilled; every output against float64 from the device's own rotated rows."""
    rng = np.random.default_rng(14)
    heads, kv, hd, page, rt = 4, 2, 80, 16, dev.rt
    hw, fused = heads + kv, (heads + 2 * kv) * hd  # a row: queries, keys, values
    rope = hip.Rope(hd, 20)
    c = hip.KVPages(cache, 2, kv, hd, page, 24)
    table = np.array([[5, 0, 11, 7, 2, 9], [1, 23, 3, 20, 8, 4]], np.int32)
    ptable, plen = dev.put(table), dev.put(np.zeros(2, np.int32))
    scale, size = hd ** -0.5, np.dtype(bits_dtype(dtype)).itemsize
    st = C.c_void_p()
    assert rt.hipStreamCreateWithFlags(C.byref(st), 1) == 0

    def slot(i, t):
        return table[i, t // page] * page + t % page

    def rows(n):
        return dev.put(encode(dtype, rng.standard_normal((n, fused)))[0])

    def turned(x, n):
        """The device's rotated rows, and what the cache holds of their keys and values."""
        v = decode(dtype, dev.get(x, (n, fused), bits_dtype(dtype)))
        return v[:, :heads * hd], v[:, heads * hd:hw * hd], v[:, hw * hd:]

    def check(got, q, ks, vs, seen, keys, rounded):
        for h in range(heads):
            g = slice(h // 2 * hd, h // 2 * hd + hd)
            want, mag, load = _attention(q[:, h * hd:h * hd + hd], ks[:, g], vs[:, g], scale, seen)
            assert np.all(np.abs(got[:, h * hd:h * hd + hd] - want) <= _tolerance(want, mag, load, keys, hd, dtype, rounded))

    w = 0 if dtype == W.F32 else EPS[dtype]
    # both prompts at once
    lens = [37, 50]
    n = sum(lens)
    x, out = rows(n), _empty(dev, dtype, n, heads * hd)
    pos = np.concatenate([np.arange(m) for m in lens]).astype(np.int32)
    slots = np.concatenate([slot(i, np.arange(m)) for i, m in enumerate(lens)]).astype(np.int32)
    off = dev.put(np.cumsum([0] + lens).astype(np.int32))
    pp, ps = dev.put(pos), dev.put(slots)
    kat, vat = x + heads * hd * size, x + hw * hd * size
    rope.rotate(dtype, x, fused, n, hw, pp, dtype, x, fused, st.value)
    c.write(1, dtype, kat, fused, vat, fused, ps, n, st.value)
    hip.attention(dtype, x, fused, heads, kat, fused, vat, fused, kv, hd, scale, True, off, off, 2, n, n, out, heads * hd, st.value)
    assert rt.hipStreamSynchronize(st) == 0
    q, k, v = turned(x, n)
    got = decode(dtype, dev.get(out, (n, heads * hd), bits_dtype(dtype)))
    held = [[], []]
    at = 0
    for i, m in enumerate(lens):
        s = slice(at, at + m)
        check(got[s], q[s], k[s], v[s], np.tri(m, dtype=bool), m, w)
        held[i] = [_held(cache, k[s], hd), _held(cache, v[s], hd)]
        at += m
    # a second chunk of the first prompt, over what is read back
    m = 21
    x, out = rows(m), _empty(dev, dtype, m, heads * hd)
    total = lens[0] + m
    ps = dev.put(slot(0, np.arange(total)).astype(np.int32))
    kr, vr = (_empty(dev, dtype, total, kv * hd) for _ in range(2))
    rope.rotate(dtype, x, fused, m, hw, dev.put(np.arange(lens[0], total, dtype=np.int32)), dtype, x, fused, st.value)
    c.write(1, dtype, x + heads * hd * size, fused, x + hw * hd * size, fused, ps + 4 * lens[0], m, st.value)
    c.read(1, dtype, kr, kv * hd, vr, kv * hd, ps, total, st.value)
    hip.attention(dtype, x, fused, heads, kr, kv * hd, vr, kv * hd, kv, hd, scale, True, dev.put(np.array([0, m], np.int32)),
                  dev.put(np.array([0, total], np.int32)), 1, m, total, out, heads * hd, st.value)
    assert rt.hipStreamSynchronize(st) == 0
    q, k, v = turned(x, m)
    held[0] = [np.concatenate([a, _held(cache, b, hd)]) for a, b in zip(held[0], (k, v))]
    back = [decode(dtype, dev.get(p, (total, kv * hd), bits_dtype(dtype))) for p in (kr, vr)]
    for a, b in zip(back, held[0]):
        assert np.array_equal(a, encode(dtype, b)[1])
    check(decode(dtype, dev.get(out, (m, heads * hd), bits_dtype(dtype))), q, *back, np.arange(total) <= np.arange(m)[:, None] + lens[0], total, w)
    lens[0] = total
    # decode steps of both from one graph
    x, out = rows(2), _empty(dev, dtype, 2, heads * hd)
    pp, ps = dev.put(np.zeros(2, np.int32)), dev.put(np.zeros(2, np.int32))
    graph, ex = C.c_void_p(), C.c_void_p()
    assert rt.hipStreamBeginCapture(st, 0) == 0
    rope.rotate(dtype, x, fused, 2, hw, pp, dtype, x, fused, st.value)
    c.write(1, dtype, x + heads * hd * size, fused, x + hw * hd * size, fused, ps, 2, st.value)
    c.attend(1, dtype, x, fused, heads, scale, ptable, 6, plen, 2, out, heads * hd, st.value)
    assert rt.hipStreamEndCapture(st, C.byref(graph)) == 0
    assert rt.hipGraphInstantiate(C.byref(ex), graph, None, None, C.c_size_t(0)) == 0
    for step in range(4):
        dev.fill(x, encode(dtype, rng.standard_normal((2, fused)))[0])
        dev.fill(pp, np.array(lens, np.int32))
        dev.fill(ps, np.array([slot(i, np.array(m)) for i, m in enumerate(lens)], np.int32))
        lens = [m + 1 for m in lens]
        dev.fill(plen, np.array(lens, np.int32))
        assert rt.hipGraphLaunch(ex, st) == 0 and rt.hipStreamSynchronize(st) == 0
        q, k, v = turned(x, 2)
        got = decode(dtype, dev.get(out, (2, heads * hd), bits_dtype(dtype)))
        for i in range(2):
            held[i] = [np.concatenate([a, _held(cache, b[i:i + 1], hd)]) for a, b in zip(held[i], (k, v))]
            check(got[i:i + 1], q[i:i + 1], *held[i], None, lens[i], _weights_rounded(cache, dtype))
    rt.hipGraphExecDestroy(ex)
    rt.hipGraphDestroy(graph)
    rt.hipStreamDestroy(st)
    c.close()
    rope.close()


def test_two_threads_and_many_streams(hip, dev):
    """Long attention of two threads on one cache, over more streams than keep scratch of their own: an idle cache's bits."""
    import threading
    rng = np.random.default_rng(15)
    heads, hd, page, length = 2, 64, 64, 4000
    width = -(-length // page)
    rows = width * page
    c = hip.KVPages(W.F16, 1, 2, hd, page, width)
    pk, ld, _ = _rows(rng, dev, W.F16, rows, 2 * hd)
    c.write(0, W.F16, pk, ld, pk, ld, dev.put(np.arange(rows, dtype=np.int32)), rows)
    table, lengths = dev.put(np.arange(width, dtype=np.int32)), dev.put(np.array([length], np.int32))
    qs = [_rows(rng, dev, W.F32, 1, heads * hd)[0] for _ in range(2)]
    y = [[dev.put(np.zeros((1, heads * hd), np.float32)) for _ in range(12)] for _ in range(2)]
    streams, errors = [C.c_void_p() for _ in range(12)], []
    for st in streams:
        assert dev.rt.hipStreamCreateWithFlags(C.byref(st), 1) == 0

    def work(i):
        try:
            for j, out in enumerate(y[i]):
                c.attend(0, W.F32, qs[i], heads * hd, heads, 0.125, table, width, lengths, 1, out, heads * hd, streams[j].value)
        except Exception as err:
            errors.append(err)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    got = [[dev.get(out, (1, heads * hd)).copy() for out in outs] for outs in y]
    for i in range(2):
        c.attend(0, W.F32, qs[i], heads * hd, heads, 0.125, table, width, lengths, 1, y[i][0], heads * hd)
        want = dev.get(y[i][0], (1, heads * hd))
        assert np.abs(want).max() > 0 and all(np.array_equal(g, want) for g in got[i])
    for st in streams:
        dev.rt.hipStreamDestroy(st)
    c.close()


def test_threads_share_a_buffer_in_turn():
    """Products of two threads that end, on a buffer that they and five streams share: again and again, since an
    order of their streams that rested on events alone was lost in one of about 100 runs."""
    import test_zz_no_alloc as products
    for _ in range(40):
        products.test_products_in_flight_on_many_streams(W.F16, 70)


def test_threads_share_the_library_array_in_turn(hip, dev):
    """No-allocation products of threads that end with their work enqueued, behind those of four streams."""
    import threading
    rng = np.random.default_rng(33)
    rows, cols, sizes = 900, 1536, (70, 73, 76, 79)
    w = hip.Weight(W.Tensor(W.F16, rows, cols, encode(W.F16, rng.standard_normal((rows, cols)))[0].reshape(-1).view(np.uint8)))
    x = [dev.put(rng.standard_normal((sizes[-1], cols)).astype(np.float32)) for _ in range(6)]
    y = [[_empty(dev, W.F32, m, rows) for m in sizes] for _ in x]
    streams = [C.c_void_p() for _ in range(4)]
    for st in streams:
        assert dev.rt.hipStreamCreateWithFlags(C.byref(st), 1) == 0

    def run(i, stream):
        dev.rt.hipSetDevice(0)
        for k, m in enumerate(sizes):
            w.mul_device_noalloc(x[i], m, y[i][k], stream)

    want = []
    for i in range(6):
        run(i, streams[0].value)
        want.append([dev.get(y[i][k], (m, rows)) for k, m in enumerate(sizes)])
    for _ in range(60):
        clear = np.full((sizes[-1], rows), np.nan, np.float32)
        for i in range(6):
            for k, m in enumerate(sizes):
                assert dev.rt.hipMemcpy(y[i][k], clear.ctypes.data, m * rows * 4, 1) == 0
        for i in range(4):
            run(i, streams[i].value)
        threads = [threading.Thread(target=run, args=(i, 2)) for i in (4, 5)]  # hipStreamPerThread
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for i in range(6):
            for k, m in enumerate(sizes):
                assert np.array_equal(dev.get(y[i][k], (m, rows)), want[i][k]), (i, m)
    for st in streams:
        dev.rt.hipStreamDestroy(st)
    w.close()


def test_refusals_of_handles(hip, dev):
    """Refusals that need an open handle; none of them reaches the device."""
    r, c = hip.Rope(64, 64), hip.KVPages(W.Q8_0, 2, 4, 64, 16, 4)
    p = dev.put(np.zeros(1 << 16, np.uint8))
    for n, heads in ((-1, 1), (1, 0), (1, -4), (1, 1 << 20)):
        with pytest.raises(hip.TinyoaiError, match="invalid rotation"):
            r.rotate(W.F32, p, 64, n, heads, p, W.F32, p + 4096, 64)
    for args, match in (((W.Q8_0, p, 64, 1, 1, p, W.F32, p, 64), "unsupported x"), ((W.F32, None, 64, 1, 1, p, W.F32, p, 64), "x is null"),
                        ((W.F32, p, 63, 1, 1, p, W.F32, p, 64), "x rows"), ((W.F32, p, 64, 1, 1, None, W.F32, p, 64), "positions"),
                        ((W.F32, p + 2, 64, 1, 1, p, W.F32, p, 64), "aligned"), ((W.F32, p, 64, 1, 1, p, W.Q8_0, p, 64), "unsupported out")):
        with pytest.raises(hip.TinyoaiError, match=match):
            r.rotate(*args)
    r.rotate(W.F32, p, 64, 0, 1, p, W.F32, p, 64)
    for call in (c.write, c.read):
        for args, match in (((2, W.F32, p, 256, p, 256, p, 1), "layer"), ((-1, W.F32, p, 256, p, 256, p, 1), "layer"),
                            ((0, W.Q8_0, p, 256, p, 256, p, 1), "unsupported k"), ((0, W.F32, p, 255, p, 256, p, 1), "k rows"),
                            ((0, W.F32, p, 256, p, 255, p, 1), "v rows"), ((0, W.F32, p, 256, None, 256, p, 1), "v is null"),
                            ((0, W.F32, p, 256, p, 256, None, 1), "slots"), ((0, W.F32, p, 256, p, 256, p, -1), "slots"),
                            ((0, W.F16, p + 1, 256, p, 256, p, 1), "aligned")):
            with pytest.raises(hip.TinyoaiError, match=match):
                call(*args)
        call(0, W.F32, p, 256, p, 256, p, 0)
    r.close()
    c.close()
    with pytest.raises(hip.TinyoaiError, match="closed"):
        r.rotate(W.F32, p, 64, 1, 1, p, W.F32, p, 64)
    with pytest.raises(hip.TinyoaiError, match="closed"):
        c.read(0, W.F32, p, 256, p, 256, p, 1)
