"""Rotary positions, the paged cache and the attention operators on the GPU where they may go wrong: the kernels' forms for
large calls."""
import numpy as np
import pytest

from experts_fixture import EPS, Device, bits_dtype, decode, encode
from test_gpu_serving import CACHES, TYPES, _attention, _empty, _held, _tolerance, _weights_rounded
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
# first, pairs of a sequence and a key head are fewer than the waves (1024 at 256 values a head, 2048 at up to 128, 3072 at
# up to 64, 4096 at up to 32), in the others more.
MANY = [(16, 8, 64, 64, 12, 2100), (32, 32, 80, 16, 96, 500), (8, 4, 256, 32, 300, 200), (360, 20, 128, 8, 60, 150),
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
