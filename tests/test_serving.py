"""Host side of the rotary positions, the paged cache and the attention operators: refusals, which make no device call."""
import ctypes as C

import pytest

from tinyoai_amd import hip
from tinyoai_amd import weights as W

A = 1 << 20  # an aligned address that nothing reads: every call here is refused


def _refused(match, call, *args, **kwargs):
    with pytest.raises(hip.TinyoaiError, match=match):
        call(*args, **kwargs)


def test_rope_open_refusals():
    for hd, rot in ((0, 0), (12, 4), (264, 8), (64, 0), (64, 66), (64, 7), (-8, 2)):
        _refused("invalid rotation", hip.Rope, hd, rot)
    for theta in (1.0, 0.0, -3.0, float("nan"), float("inf")):
        _refused("invalid rotary base", hip.Rope, 64, 64, theta=theta)
    for factor in (0.5, 0.0, float("nan"), float("inf")):
        _refused("invalid rotary factor", hip.Rope, 64, 64, scaling="linear", factor=factor)
    for context, low, high in ((0, 1, 4), (8192, 0, 4), (8192, 4, 4), (8192, 4, 1), (8192, 1, float("inf")),
                               (8192, float("nan"), 4)):
        for scaling in ("bands", "yarn"):
            _refused("invalid rotary scaling", hip.Rope, 64, 64, scaling=scaling, factor=8.0, context=context, low=low, high=high)
    L, out = hip.lib(), C.c_void_p()
    ok = [64, 64, 0, 0, 1e4, 1.0, 0, 0.0, 0.0]
    for at, value, match in ((2, 2, b"layout"), (3, 4, b"scaling"), (3, -1, b"scaling")):
        c = hip.RopeConfig(*[value if i == at else x for i, x in enumerate(ok)])
        assert L.tinyoai_rope_open(C.byref(c), C.byref(out)) == -1 and match in L.tinyoai_last_error()
    assert L.tinyoai_rope_open(None, C.byref(out)) == -1
    assert L.tinyoai_rope_open(C.byref(hip.RopeConfig(*ok)), None) == -1


def test_closed_handles():
    L = hip.lib()
    assert L.tinyoai_rope_device(None, 0, A, 64, 1, 1, A, 0, A, 64, None) == -1 and b"closed" in L.tinyoai_last_error()
    assert L.tinyoai_kv_pages_write_device(None, 0, 0, A, 64, A, 64, A, 1, None) == -1
    assert L.tinyoai_kv_pages_read_device(None, 0, 0, A, 64, A, 64, A, 1, None) == -1
    assert L.tinyoai_kv_pages_attend_device(None, 0, 0, A, 64, 1, 1.0, A, 1, A, 1, A, 64, None) == -1
    assert b"closed" in L.tinyoai_last_error()
    assert L.tinyoai_rope_close(None) == 0 and L.tinyoai_kv_pages_close(None) == 0


def test_kv_pages_open_refusals():
    for t in (W.MXFP4, 7, -1):
        _refused("unsupported paged cache type", hip.KVPages, t, 1, 8, 64, 16, 4)
    for layers, heads, hd in ((0, 8, 64), (1, 0, 64), (1, 8, 0), (1, 8, 20), (1, 8, 264), (1, 1 << 20, 64), (-1, 8, 64)):
        _refused("invalid paged cache of", hip.KVPages, W.F16, layers, heads, hd, 16, 4)
    for page, pages in ((0, 4), (12, 4), (2048, 4), (-16, 4), (16, 0), (16, -1), (1024, (1 << 20) + 1)):
        _refused("invalid paged cache of", hip.KVPages, W.F16, 1, 8, 64, page, pages)
    _refused("bytes", hip.KVPages, W.F32, 1 << 20, 1 << 14, 256, 1024, 1 << 20)
    assert hip.lib().tinyoai_kv_pages_open(W.F16, 1, 8, 64, 16, 4, None) == -1


def test_attention_refusals():
    def call(dtype=W.F16, q=A, ldq=512, heads=8, k=A, ldk=256, v=A, ldv=256, kv_heads=4, hd=64, scale=0.125, qo=A, ko=A,
             sequences=2, nq=10, nk=10, out=A, ldo=512):
        hip.attention(dtype, q, ldq, heads, k, ldk, v, ldv, kv_heads, hd, scale, True, qo, ko, sequences, nq, nk, out, ldo)

    for hd in (0, -8, 60, 264):
        _refused("unsupported head width", call, hd=hd)
    for heads, kv in ((8, 3), (0, 4), (8, 0), (-8, 4), (1 << 20, 4)):
        _refused("query heads over", call, heads=heads, kv_heads=kv)
    for t in (W.Q8_0, W.MXFP4, -1):
        _refused("unsupported q type", call, dtype=t)
    for name in ("q", "k", "v", "out"):
        _refused(f"{name} is null", call, **{name: None})
        _refused(f"{name} is not aligned", call, **{name: A + 1})
    for name, what in (("ldq", "q"), ("ldk", "k"), ("ldv", "v"), ("ldo", "out")):
        _refused(f"{what} rows of", call, **{name: 255})
        _refused(f"{what} rows are", call, **{name: (1 << 22) + 1})
    for scale in (float("nan"), float("inf")):
        _refused("invalid scale", call, scale=scale)
    for bad in (dict(qo=None), dict(ko=None), dict(sequences=0), dict(nq=-1), dict(nk=-1), dict(nq=(1 << 30) + 1),
                dict(nk=(1 << 30) + 1)):
        _refused("invalid offsets", call, **bad)
    _refused("exceed", call, nq=1 << 30)
    _refused("exceed", call, nq=1 << 21, sequences=1 << 21)
    call(nq=0)  # nothing to do


def test_attention_of_nothing():
    """No queries: nothing to do, whatever is empty with them. Refusals stay."""
    def call(q=None, k=None, v=None, qo=None, ko=None, sequences=0, nq=0, nk=0, out=None):
        hip.attention(W.F16, q, 512, 8, k, 256, v, 256, 4, 64, 0.125, True, qo, ko, sequences, nq, nk, out, 512)

    call()
    call(nk=5)
    call(sequences=3, qo=A, ko=A)
    _refused("invalid offsets", call, sequences=-1)
    _refused("invalid offsets", call, nk=-1)
    _refused("q is null", call, nq=1, qo=A, ko=A, sequences=1)
    _refused("out is null", call, nq=1, qo=A, ko=A, sequences=1, q=A)
    _refused("k is null", call, nq=1, nk=1, qo=A, ko=A, sequences=1, q=A, out=A)
    _refused("v is null", call, nq=1, nk=1, qo=A, ko=A, sequences=1, q=A, out=A, k=A)
