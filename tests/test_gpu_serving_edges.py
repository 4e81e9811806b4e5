"""Rotary positions, the paged cache and the attention operators on the GPU where they may go wrong: the kernels' forms for
large calls, values that are not finite, weights that are small, no rows."""
import numpy as np
import pytest

from experts_fixture import EPS, Device, bits_dtype, decode, encode
from test_gpu_serving import CACHES, TYPES, U, _attention, _empty, _encoded, _held, _rope_check, _rows, _take, _tolerance, _weights_rounded
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


# ---------------------------------------------------------------- new tokens: more work than a launch has waves
# (query heads, key heads, head width, page, sequences, longest): a wave's run holds several pairs or pieces of them. In the
# first, pairs of a sequence and a key head are fewer than the waves (four blocks of four a CU at up to 32 values a head,
# three at up to 64, two at up to 128, two of two waves at 256), in the others more.
MANY = [(16, 8, 64, 64, 12, 2100), (32, 32, 80, 16, 95, 500), (8, 4, 256, 32, 300, 200), (360, 20, 128, 8, 60, 150),
        (64, 32, 64, 64, 100, 300), (32, 32, 24, 4, 130, 90)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cache", CACHES)
def test_attend_many_pairs(hip, dev, cache, dtype):
    """Each call follows one of other lengths on the same handle and stream, whose records lie in the scratch."""
    rng = np.random.default_rng(31)
    for heads, kv, hd, page, n, longest in MANY:
        pages, width = 96, -(-6000 // page)
        rows = pages * page
        (_, k), (_, v) = (encode(W.F32, rng.standard_normal((rows, kv * hd))) for _ in range(2))
        c = hip.KVPages(cache, 1, kv, hd, page, pages)
        c.write(0, W.F32, dev.put(k.astype(np.float32)), kv * hd, dev.put(v.astype(np.float32)), kv * hd,
                dev.put(np.arange(rows, dtype=np.int32)), rows)
        table = rng.integers(0, pages, (n, width)).astype(np.int32)  # (requests share pages)
        lengths = rng.integers(longest // 2 if n == 12 else 0, longest, n).astype(np.int32)
        if n > 12:
            lengths[rng.permutation(n)[:10]] = [0, 1, 31, 32, 33, 0, 64, 65, 127, 0]
            lengths[n // 3] = 6000
        qb, q = encode(dtype, rng.standard_normal((n, heads * hd)))
        out, pq, pt = _empty(dev, dtype, n, heads * hd), dev.put(qb), dev.put(table)
        for x in (lengths[::-1] // 2 + 7, lengths):
            c.attend(0, dtype, pq, heads * hd, heads, hd ** -0.5, pt, width, dev.put(np.ascontiguousarray(x)), n, out, heads * hd)
        got = decode(dtype, dev.get(out, (n, heads * hd), bits_dtype(dtype))).reshape(n, kv, heads // kv, hd)
        q = q.reshape(n, kv, heads // kv, hd)
        k, v = (_held(cache, x, hd).reshape(rows, kv, hd) for x in (k, v))
        for i, x in enumerate(lengths):
            t = np.arange(x)
            slots = table[i, t // page] * page + t % page
            ks, vs = k[slots].transpose(1, 0, 2), v[slots].transpose(1, 0, 2)
            for g in range(kv):
                want, mag, load = _attention(q[i, g], ks[g], vs[g], hd ** -0.5)
                tol = _tolerance(want, mag, load, int(x), hd, dtype, _weights_rounded(cache, dtype))
                assert np.all(np.abs(got[i, g] - want) <= tol), (heads, kv, hd, i, g, x)
        c.close()
        dev.close()


# ---------------------------------------------------------------- values that are not finite
def _softmax_sums(q, k, v, scale, seen=None):
    """The attention's formula in float64 with IEEE rules for infinities and NaN, of queries [m, hd]: (outputs, and of the
    finite values alone the sums of weight times magnitude and the largest sums of scale |q| |k|)."""
    with np.errstate(invalid="ignore", over="ignore"):
        s = (q[:, None] * k).sum(-1) * scale
        if seen is not None:
            s = np.where(seen, s, -np.inf)
        top = s.max(-1, keepdims=True)
        p = np.exp(s - top)
        p = p / p.sum(-1, keepdims=True)
        terms = p[..., None] * v
        if seen is not None:  # what is not seen has no effect, whatever it holds
            terms = np.where(seen[..., None], terms, 0)
        out = terms.sum(1)
    mag = np.where(np.isfinite(terms), np.abs(terms), 0).sum(1)
    load = np.where(np.isfinite(k), np.abs(q[:, None] * k), 0).sum(-1).max(-1, initial=0)[:, None] * abs(scale)
    if seen is not None:
        out[~seen.any(-1)] = 0
    return out, mag, load


def _same(got, want, tol):
    """Where the formula's result is finite within the tolerance, else that result."""
    assert np.array_equal(np.isnan(got), np.isnan(want)), (np.isnan(got).sum(), np.isnan(want).sum())
    at = np.isfinite(want)
    assert np.array_equal(got[~at], want[~at], equal_nan=True)
    assert np.all(np.abs(got[at] - want[at]) <= np.broadcast_to(tol, want.shape)[at])


def _infinite_attend(hip, dev, rng, cache, dtype, heads, kv, hd, page, lengths, spoil):
    """New tokens over pages whose rows `spoil(i, k, v, q)` has changed, [length, kv, hd] of sequence i (q [heads, hd])."""
    n, width = len(lengths), -(-max(lengths) // page)
    pages, rows = n * width, n * width * page
    table = rng.permutation(pages).astype(np.int32).reshape(n, width)
    qb, q = encode(dtype, rng.standard_normal((n, heads * hd)))
    k, v = (rng.standard_normal((rows, kv, hd)).astype(np.float32) for _ in range(2))
    slots = [table[i, np.arange(x) // page] * page + np.arange(x) % page for i, x in enumerate(lengths)]
    for i, s in enumerate(slots):
        ks, vs = k[s], v[s]
        spoil(i, ks, vs, q[i].reshape(heads, hd))
        k[s], v[s] = ks, vs
    c = hip.KVPages(cache, 1, kv, hd, page, pages)
    c.write(0, W.F32, dev.put(k), kv * hd, dev.put(v), kv * hd, dev.put(np.arange(rows, dtype=np.int32)), rows)
    out = _empty(dev, dtype, n, heads * hd)
    scale = hd ** -0.5
    c.attend(0, dtype, dev.put(qb), heads * hd, heads, scale, dev.put(table), width, dev.put(np.asarray(lengths, np.int32)), n, out,
             heads * hd)
    got = decode(dtype, dev.get(out, (n, heads * hd), bits_dtype(dtype))).reshape(n, heads, hd)
    c.close()
    with np.errstate(invalid="ignore", over="ignore"):
        k, v = (_held(cache, x.reshape(rows, -1).astype(np.float64), hd).reshape(rows, kv, hd) for x in (k, v))
    for i, s in enumerate(slots):
        for h in range(heads):
            g = h // (heads // kv)
            want, mag, load = _softmax_sums(q[i].reshape(heads, hd)[h:h + 1], k[s, g], v[s, g], scale)
            with np.errstate(invalid="ignore"):
                tol = _tolerance(np.where(np.isfinite(want), want, 0), mag, load, lengths[i], hd, dtype, _weights_rounded(cache, dtype))
            _same(got[i, h], want[0], tol[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cache", TYPES)
def test_attend_infinities(hip, dev, cache, dtype):
    """Infinities that are seen count as fp32 sums of products have them: one in the values makes its outputs infinite, both
    signs NaN; one in the keys weighs nothing where the score falls to -inf and makes NaN where it rises to +inf."""
    rng = np.random.default_rng(41)

    def values(i, k, v, q):
        v[rng.integers(0, len(v), 5), :, rng.integers(0, v.shape[2], 5)] = np.inf
        v[rng.integers(0, len(v), 5), :, rng.integers(0, v.shape[2], 5)] = -np.inf

    def one_value(i, k, v, q):  # its weight is exactly 1
        v[0, :, ::3] = np.inf

    def keys(i, k, v, q):  # a score of -inf for the first head of each key head
        group = len(q) // k.shape[1]
        for g in range(k.shape[1]):
            for t in rng.integers(0, len(k), 3):
                d = rng.integers(0, k.shape[2])
                k[t, g, d] = -np.inf * np.sign(q[g * group, d])

    def both(i, k, v, q):
        if i == 0:
            values(i, k, v, q)
        if i == 1:
            keys(i, k, v, q)

    for heads, kv, hd, page, lengths, spoil in ((4, 2, 64, 16, (40, 3, 200), values), (4, 2, 64, 16, (1, 2), one_value),
                                                (2, 2, 80, 8, (33, 150), values), (3, 1, 128, 64, (65, 7), keys),
                                                (2, 2, 96, 32, (31, 100), keys), (20, 1, 40, 4, (50, 9), both),
                                                (2, 1, 256, 16, (70, 20), both), (1, 1, 8, 1, (9, 40), values),
                                                (4, 4, 128, 16, (3000, 2500, 1000), both), (2, 1, 64, 64, (6000, 5000), both)):
        _infinite_attend(hip, dev, rng, cache, dtype, heads, kv, hd, page, lengths, spoil)


# ---------------------------------------------------------------- small weights
@pytest.mark.parametrize("dtype", [W.F16, W.BF16])
@pytest.mark.parametrize("heads,hd,nq,nk,causal", [(1, 64, 1, 131072, False), (1, 128, 1, 1 << 20, False), (2, 80, 130, 20000, True),
                                                   (1, 64, 19, 1500, False), (2, 96, 50, 1500, True), (16, 128, 2048, 2048, True),
                                                   (64, 64, 2048, 2048, True), (8, 256, 4096, 4096, False)])
def test_prompt_small_weights(hip, dev, dtype, heads, hd, nq, nk, causal):
    """One key far above all others, whose weights count together: 17.4 nats below it each, or spread over 25 nats."""
    rng = np.random.default_rng(51)
    for scores in (np.full(nk, -17.4), -25 * rng.random(nk)):
        scores[0] = 0  # (the causal queries all see it)
        k = np.zeros((nk, hd))
        k[:, 0] = scores
        v = rng.random((nk, hd))
        v[0, ::2] = 0
        kb, k = encode(dtype, k)
        vb, v = encode(dtype, v)
        q = np.zeros((nq, heads, hd), np.float32)
        q[..., 0] = 1
        qb = encode(dtype, q.reshape(nq, -1))[0]
        out = _empty(dev, dtype, nq, heads * hd)
        hip.attention(dtype, dev.put(qb), heads * hd, heads, dev.put(kb), hd, dev.put(vb), hd, 1, hd, 1.0, causal,
                      dev.put(np.array([0, nq], np.int32)), dev.put(np.array([0, nk], np.int32)), 1, nq, nk, out, heads * hd)
        got = decode(dtype, dev.get(out, (nq, heads * hd), bits_dtype(dtype))).reshape(nq, heads, hd)
        p = np.exp(k[:, 0])
        last = np.arange(nq) + nk - nq if causal else np.full(nq, nk - 1)
        top, total, keys = np.cumsum(p[:, None] * v, 0)[last], np.cumsum(p)[last][:, None], last[:, None] + 1
        want = top / total
        # a weight, of at most 1, rounds by half a step (and its score by 25 U, its power by 2 U); fp16's are multiples of
        # 2^-35 of the largest at least, and then off by 2^-36 each; the sums have chains of keys / 4 terms
        tiny = keys * (2.0 ** -36 if dtype == W.F16 else 0)
        off = EPS[dtype] + 30 * U + 2 * (keys / 4 + 64) * U
        tol = 1.01 * (2 * off * want + (1 + want) * tiny / total) + EPS[dtype] * want + (2.0 ** -25 if dtype == W.F16 else 0)
        assert np.all(np.abs(got - want[:, None]) <= tol[:, None]), (np.abs(got - want[:, None]) / tol[:, None]).max()
        dev.close()


# ---------------------------------------------------------------- empty buffers
def test_calls_of_nothing(hip, dev):
    """Empty arrays have no address: calls without rows do nothing, and queries over no keys give zeros."""
    r, c = hip.Rope(64, 64), hip.KVPages(W.F16, 1, 4, 64, 16, 4)
    r.rotate(W.F32, 0, 256, 0, 4, 0, W.F32, 0, 256)
    r.rotate(W.F32, 0, 256, 0, 4, 0, W.F16, 0, 256)
    for call in (c.write, c.read):
        call(0, W.F32, 0, 256, 0, 256, 0, 0)
    c.attend(0, W.F32, 0, 256, 4, 0.125, 0, 0, 0, 0, 0, 256)
    for dtype in TYPES:
        for nq in (1, 50, 700):
            q = dev.put(np.ones((nq, 256), bits_dtype(dtype)))
            qo, ko = dev.put(np.array([0, nq // 2, nq], np.int32)), dev.put(np.zeros(3, np.int32))
            for causal in (True, False):
                out = _empty(dev, dtype, nq, 256)
                hip.attention(dtype, q, 256, 4, 0, 256, 0, 256, 4, 64, 0.125, causal, qo, ko, 2, nq, 0, out, 256)
                assert not dev.get(out, (nq, 256), bits_dtype(dtype)).any()
    r.close()
    c.close()


# ---------------------------------------------------------------- prompts of ordinary size
def _form(dtype, heads, hd, nq, nk, sequences):
    """(groups of 32 queries of a block, groups of keys, parts of the keys, sets of queries a wave) as launch_prompt chooses."""
    def tiles(queries):
        return nq // queries + min(sequences, nq)

    blocks, keys = tiles(128) * heads, nk // max(1, min(sequences, nk))
    sets = 2 if dtype != W.F32 and hd <= 64 and tiles(256) * heads >= 512 else 1
    if blocks >= 256:
        return 4, 1, 1, sets
    if dtype == W.F32:
        groups = 2 if hd > 128 else 4
        return 1, groups, max(1, min(512 // (tiles(32) * heads), -(-keys // (32 * groups)))), 1
    if keys >= 2048:
        return 4, 1, max(1, min(512 // blocks, keys // 1024)), sets
    return (1, 4, 1, 1) if nq <= 32 else (2, 4, 1, 1) if hd <= 128 else (4, 1, 1, sets)


def _prompt_rows(hip, dev, rng, dtype, heads, kv, hd, lengths, causal, pad=0, shift=0, hidden=False, spread=1.0):
    """Sequences of (queries, keys), checked at rows around the tiles' borders and some others, of three heads."""
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
        if not m:
            continue
        rows = np.concatenate([np.arange(0, m, 32), np.arange(31, m, 32), [m - 1], rng.integers(0, m, 12)])
        rows = np.unique(np.concatenate([rng.permutation(rows)[:30], [0, m - 1, max(m - keys, 0), max(m - keys - 1, 0)]]))
        rows = rows[rows < m]
        seen = np.arange(keys) <= rows[:, None] + keys - m if causal else np.ones((len(rows), keys), bool)
        for h in {0, heads - 1, int(rng.integers(0, heads))}:
            g = slice(h // (heads // kv) * hd, h // (heads // kv) * hd + hd)
            qs, ks, vs = q[q0 + rows, h * hd:h * hd + hd], k[k0:k0 + keys, g], v[k0:k0 + keys, g]
            bad_k, bad_v = ~np.isfinite(ks).all(-1), ~np.isfinite(vs)
            want, mag, load = _attention(qs, np.where(np.isfinite(ks), ks, 0), np.where(bad_v, 0, vs), scale, seen)
            fine = ~((seen @ bad_k.astype(float))[:, None] + seen @ bad_v.astype(float) > 0)
            with np.errstate(invalid="ignore"):  # (a score of -inf is a weight of zero: such a key need not show)
                zero = (seen & (qs @ ks.T == -np.inf)).any(-1) if bad_k.any() else np.zeros(len(rows), bool)
            part = got[q0 + rows, h]
            assert not np.isfinite(part[~fine & ~zero[:, None]]).any()
            tol = _tolerance(want, mag, load, keys, hd, dtype, 0 if dtype == W.F32 else EPS[dtype])
            assert np.all((np.abs(part - want) <= tol) | ~fine), (m, keys, h)
            if causal and m > keys:
                assert not part[rows < m - keys].any()


LARGE = ((1500, 1500), (37, 37), (1, 700), (0, 5), (2000, 2000), (700, 500), (300, 1500), (260, 0))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,heads,kv,hd,sets", [(t, h, kv, hd, sets) for t, shapes in (
    (W.F16, ((32, 8, 64, 2), (32, 32, 8, 2), (32, 1, 40, 2), (8, 2, 64, 1), (8, 8, 80, 1), (8, 4, 96, 1), (8, 2, 128, 1), (8, 1, 256, 1), (8, 2, 72, 1))),
    (W.BF16, ((32, 8, 64, 2), (32, 4, 24, 2), (32, 2, 40, 2), (8, 2, 32, 1), (8, 8, 80, 1), (8, 4, 96, 1), (8, 2, 128, 1), (8, 1, 200, 1))),
    (W.F32, ((8, 2, 8, 1), (8, 1, 64, 1), (8, 8, 80, 1), (8, 2, 96, 1), (8, 2, 128, 1), (8, 4, 256, 1), (8, 4, 160, 1)))) for h, kv, hd, sets in shapes])
def test_prompt_large(hip, dev, dtype, heads, kv, hd, sets, causal):
    """Blocks of 128 or 256 queries that see all of their keys: ragged sequences, more queries than keys and none, rows at
    16-byte distances and at odd ones, values that are not finite in what some do not see."""
    rng = np.random.default_rng(71)
    nq, nk = (sum(x[i] for x in LARGE) + 2 for i in range(2))
    assert _form(dtype, heads, hd, nq, nk, len(LARGE)) == (4, 1, 1, sets)
    odd = dict(pad=3, shift=2 if dtype != W.F32 else 4)
    _prompt_rows(hip, dev, rng, dtype, heads, kv, hd, LARGE, causal)
    dev.close()
    _prompt_rows(hip, dev, rng, dtype, heads, kv, hd, LARGE, causal, **odd, hidden=causal)
    dev.close()
    if causal:
        _prompt_rows(hip, dev, rng, dtype, heads, kv, hd, LARGE, True, hidden=True, spread=2.0)
        dev.close()


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_small_forms(hip, dev, dtype):
    """The forms of few queries at the widths that other tests leave out."""
    rng = np.random.default_rng(72)
    for heads, kv, hd, lengths, form in ((2, 1, 96, ((20, 300),), (1, 4, 1, 1)), (2, 1, 96, ((90, 300),), (2, 4, 1, 1)),
                                         (1, 1, 96, ((90, 5000),), (4, 1, 4, 1)), (1, 1, 32, ((130, 9000),), (4, 1, 8, 1)),
                                         (2, 2, 160, ((100, 300),), (4, 1, 1, 1)), (2, 2, 256, ((9, 700),), (1, 4, 1, 1)),
                                         (3, 1, 40, ((70, 1100), (5, 9)), (2, 4, 1, 1))):
        nq, nk = (sum(x[i] for x in lengths) + 2 for i in range(2))
        assert dtype == W.F32 or _form(dtype, heads, hd, nq, nk, len(lengths)) == form
        for causal in (True, False):
            _prompt_rows(hip, dev, rng, dtype, heads, kv, hd, lengths, causal)
            _prompt_rows(hip, dev, rng, dtype, heads, kv, hd, lengths, causal, pad=1, shift=4, hidden=causal)
        dev.close()


# ---------------------------------------------------------------- many rows
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype,odtype", [(W.F32, W.F32), (W.BF16, W.BF16), (W.F16, W.F32)])
def test_rope_many_rows(hip, dev, dtype, odtype, layout):
    """Blocks of several rows, the last of fewer, few heads and many, also in place."""
    rng = np.random.default_rng(81)
    for n, heads, hd, rot, pad, shift in ((2047, 3, 64, 64, 0, 0), (2048, 5, 80, 20, 8, 0), (3001, 2, 128, 128, 1, 4), (8195, 1, 8, 2, 0, 0),
                                          (8195, 3, 72, 36, 3, 4), (5000, 2, 256, 250, 0, 0), (4099, 20, 64, 2, 0, 0)):
        positions = rng.integers(0, 100000, n)
        _rope_check(hip, dev, rng, n, heads, hd, rot, layout, dtype, odtype, positions, pad=pad, shift=shift)
        if dtype == odtype:
            px, ld, _ = _rows(rng, dev, dtype, n, heads * hd, pad, shift)
            raw = dev.get(px, (n, ld), bits_dtype(dtype)).copy()
            out, pp = dev.put(raw, shift), dev.put(positions.astype(np.int32))
            r = hip.Rope(hd, rot, layout)
            r.rotate(dtype, px, ld, n, heads, pp, dtype, out, ld)
            r.rotate(dtype, px, ld, n, heads, pp, dtype, px, ld)
            r.close()
            got = dev.get(px, (n, ld), bits_dtype(dtype))
            assert np.array_equal(got, dev.get(out, (n, ld), bits_dtype(dtype))) and not np.array_equal(got, raw)
        dev.close()


@pytest.mark.parametrize("cache,dtype", [(W.F32, W.F32), (W.F16, W.F32), (W.BF16, W.BF16), (W.Q8_0, W.F32), (W.Q8_0, W.F16)])
def test_cache_many_rows(hip, dev, cache, dtype):
    """Four rows a thread and a rest, side by side in a block and over two blocks: bit for bit, as in test_cache_rows."""
    rng = np.random.default_rng(82)
    for n, heads, hd, page, pad in ((12500, 8, 64, 16, 0), (1801, 30, 136, 64, 5), (6001, 3, 72, 1024, 1)):
        width, pages = heads * hd, -(-(n + 9) // page) + 1
        c = hip.KVPages(cache, 1, heads, hd, page, pages)
        (kb, k), (vb, v) = (_encoded(dtype, rng.standard_normal((n, width + pad)) * np.exp(rng.standard_normal(width + pad))) for _ in range(2))
        slots = rng.permutation(pages * page)[:n].astype(np.int32)
        gone = rng.random(n) < 0.05
        slots[gone] = rng.choice([-1, pages * page, -(1 << 31)], gone.sum())
        ps = dev.put(slots)
        c.write(0, dtype, dev.put(kb), width + pad, dev.put(vb), width + pad, ps, n)
        ko, vo = _empty(dev, W.F32, n, width, pad), _empty(dev, W.F32, n, width, pad)
        c.read(0, W.F32, ko, width + pad, vo, width + pad, ps, n)
        for out, x in ((ko, k), (vo, v)):
            want = np.where(gone[:, None], 0, _held(cache, x[:, :width], hd))
            assert np.array_equal(_take(dev, out, W.F32, n, width, pad), want.astype(np.float32))
        rest = np.setdiff1d(np.arange(pages * page), slots).astype(np.int32)
        ko, vo = (_empty(dev, W.F32, len(rest), width) for _ in range(2))
        c.read(0, W.F32, ko, width, vo, width, dev.put(rest), len(rest))
        assert not dev.get(ko, (len(rest), width)).any() and not dev.get(vo, (len(rest), width)).any()
        c.close()
        dev.close()
