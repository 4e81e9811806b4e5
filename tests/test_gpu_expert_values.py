"""Values of the expert products where their arithmetic could go wrong, on the GPU against float64."""
import numpy as np
import pytest

from experts_fixture import Device, encode, silu
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
