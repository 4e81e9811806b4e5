"""Host side of the mixture-of-experts operators: refusals, which make no
device call, and the encodings."""
import numpy as np
import pytest

from experts_fixture import mx_quantize, mx_values
from tinyoai_amd import hip
from tinyoai_amd import weights as W

A = 1 << 20  # an aligned address that nothing reads: every call here is refused


def _refused(match, call, *args):
    with pytest.raises(hip.TinyoaiError, match=match):
        call(*args)


def test_mxfp4_encoding():
    codes = np.arange(64, dtype=np.uint8).reshape(1, 64) % 16
    raw = W.encode_mxfp4(codes, np.array([[7, 200]], np.uint8)).reshape(2, 17)
    assert raw[0, 0] == 7 and raw[1, 0] == 200
    assert raw[0, 1] == codes[0, 0] | codes[0, 16] << 4 and raw[1, 16] == codes[0, 47] | codes[0, 63] << 4
    assert W.nbytes(W.MXFP4, 3, 64) == 3 * 34
    assert hip.mxfp4_row_bytes(32) == (64, 4) and hip.mxfp4_row_bytes(160) == (128, 8)


def test_mxfp4_statement():
    """The tests' own quantisation at values worked out by hand: a largest
    value of 6.9 scales by 1; halfway points go to even codes."""
    x = np.zeros((1, 32))
    x[0, :12] = [6.9, -.25, .75, 1.25, 1.75, 2.5, -3.5, 5, 5.01, .26, 0, -6]
    codes, scales = mx_quantize(x)
    assert scales[0, 0] == 127
    assert mx_values(codes, scales)[0, :12].tolist() == [6, 0, 1, 1, 2, 2, -4, 4, 6, .5, 0, -6]


def test_quantize_refusals():
    q, d = hip.quantize_mxfp4, hip.dequantize_mxfp4
    for n, cols in ((0, 32), (-1, 32), (1, 0), (1, 31), (1, 48), (1 << 31, 32)):
        _refused("invalid MXFP4 shape", q, W.F32, A, 64, n, cols, A, A)
        _refused("invalid MXFP4 shape", d, A, A, n, cols, W.F32, A, 64)
    for t in (W.Q8_0, W.MXFP4, -1):
        _refused("unsupported x type", q, t, A, 32, 1, 32, A, A)
        _refused("unsupported out type", d, A, A, 1, 32, t, A, 32)
    _refused("x is null", q, W.F32, None, 32, 1, 32, A, A)
    _refused("rows of 32 values are 31 apart", q, W.F32, A, 31, 1, 32, A, A)
    _refused("aligned to its type", q, W.F32, A + 2, 32, 1, 32, A, A)
    _refused("aligned to its type", d, A, A, 1, 32, W.BF16, A + 1, 32)
    _refused("invalid MXFP4 rows", q, W.F32, A, 32, 1, 32, None, A)
    _refused("invalid MXFP4 rows", d, A, None, 1, 32, W.F32, A, 32)
    _refused("16-byte", q, W.F32, A, 32, 1, 32, A + 8, A)
    _refused("16-byte", q, W.F32, A, 32, 1, 32, A, A + 2)


def test_route_refusals():
    def call(dtype=W.F32, ptr=A, ld=64, n=4, experts=64, k=2, out=(A,) * 5):
        hip.route(dtype, ptr, ld, n, experts, k, False, *out)

    for bad in (dict(n=0), dict(experts=0), dict(experts=1025, ld=2048), dict(k=0), dict(k=33), dict(k=5, experts=4),
                dict(n=1 << 30)):
        with pytest.raises(hip.TinyoaiError, match="invalid routing"):
            call(**bad)
    with pytest.raises(hip.TinyoaiError, match="unsupported logits type"):
        call(dtype=W.Q8_0)
    with pytest.raises(hip.TinyoaiError, match="63 apart"):
        call(ld=63)
    for i in range(5):
        with pytest.raises(hip.TinyoaiError, match="invalid routing outputs"):
            call(out=tuple(None if j == i else A for j in range(5)))


def test_combine_refusals():
    def call(dtype=W.F32, y=A, ldy=8, y_rows=4, pos=A, w=A, n=2, k=2, cols=8, odtype=W.F32, out=A, ldo=8):
        hip.combine(dtype, y, ldy, y_rows, pos, w, n, k, cols, odtype, out, ldo)

    for bad in (dict(n=0), dict(k=0), dict(cols=0), dict(y_rows=-1), dict(n=1 << 30)):
        with pytest.raises(hip.TinyoaiError, match="invalid sum"):
            call(**bad)
    for bad, match in ((dict(dtype=3), "unsupported y"), (dict(odtype=3), "unsupported out"), (dict(ldy=7), "7 apart"),
                       (dict(ldo=7), "7 apart"), (dict(pos=None), "positions"), (dict(w=None), "weights"),
                       (dict(out=None), "out is null"), (dict(y=A + 1), "aligned")):
        with pytest.raises(hip.TinyoaiError, match=match):
            call(**bad)


def test_expert_upload_refusals():
    L, h = hip.lib(), __import__("ctypes").c_void_p()
    a = np.zeros(64, np.uint8)

    def call(dtype=W.BF16, experts=1, rows=4, cols=8, nbytes=64, data=a.ctypes.data):
        hip.check(L.tinyoai_experts_upload(dtype, experts, rows, cols, data, None, nbytes, h))

    for bad in (dict(experts=0), dict(experts=65536), dict(rows=0), dict(rows=(1 << 28) + 1), dict(cols=0),
                dict(cols=(1 << 22) + 1)):
        _refused("invalid matrix shape", call, *[{**dict(dtype=W.BF16, experts=1, rows=4, cols=8), **bad}[k]
                                                 for k in ("dtype", "experts", "rows", "cols")])
    _refused("unsupported expert tensor type", call, W.F32)
    _refused("whole quant blocks", call, W.MXFP4, 1, 4, 48)
    _refused("need 64 bytes", call, W.BF16, 1, 4, 8, 63)
    # (2^51 bytes each: their sum does not fit 64 bits)
    _refused("bytes", call, W.BF16, 1 << 13, 1 << 28, 1 << 22, 0)
    _refused("invalid expert upload", call, W.BF16, 1, 4, 8, 64, None)


def test_absent_handles():
    L = hip.lib()
    assert L.tinyoai_weight_mul_mxfp4_device(None, A, A, 1, A, None) == -1
    assert L.tinyoai_experts_mul_device(None, W.F32, A, None, 8, 1, A, None, 1, W.F32, A, 8, None) == -1
    assert L.tinyoai_experts_free(None) == 0
    with pytest.raises(hip.TinyoaiError, match="8 and 6 bytes"):
        hip.Experts(W.BF16, 1, 2, 2, np.zeros(8, np.uint8), np.zeros(6, np.uint8))
