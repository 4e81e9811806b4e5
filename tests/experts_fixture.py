"""Device buffers and float64 statements for the mixture-of-experts tests.

Buffers come from the HIP runtime that the library is linked against (torch
bundles another one). MXFP4 is stated here by nearest values, apart from the
kernels' comparisons."""
import ctypes as C

import numpy as np

from tinyoai_amd import weights as W

GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
EPS = {W.F32: 2.0 ** -24, W.F16: 2.0 ** -11, W.BF16: 2.0 ** -8}  # half a step, relative
WIDTH = {W.F32: 4, W.F16: 2, W.BF16: 2}


class Device:
    """hipMalloc'd buffers, each with `guard` bytes before and after that must stay as they were."""
    GUARD = 512

    def __init__(self):
        from tinyoai_amd import hip
        hip.lib()  # loads libamdhip64 as the library's dependency
        self.rt = C.CDLL("libamdhip64.so.7")
        self.rt.hipMalloc.argtypes = [C.POINTER(C.c_void_p), C.c_size_t]
        self.rt.hipMemcpy.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int]
        self.rt.hipFree.argtypes = [C.c_void_p]
        self.rt.hipDeviceSynchronize.argtypes = []
        self.bufs = {}

    def put(self, a, shift=0):
        """A device copy of `a` (`shift` bytes past a 256-byte boundary)."""
        a = np.ascontiguousarray(a)
        p = C.c_void_p()
        n = a.nbytes + 2 * self.GUARD + 256
        assert self.rt.hipMalloc(C.byref(p), n) == 0
        whole = np.full(n, 0xA5, np.uint8)
        at = self.GUARD + shift
        whole[at:at + a.nbytes] = a.reshape(-1).view(np.uint8)
        assert self.rt.hipMemcpy(p, whole.ctypes.data, n, 1) == 0
        self.bufs[p.value + at] = (p.value, at, n)
        return p.value + at

    def room(self, nbytes):
        """A buffer whose bytes are not set."""
        p = C.c_void_p()
        assert self.rt.hipMalloc(C.byref(p), nbytes) == 0
        self.bufs[p.value] = (p.value, 0, nbytes)
        return p.value

    def fill(self, ptr, a):
        a = np.ascontiguousarray(a)
        assert self.rt.hipMemcpy(ptr, a.ctypes.data, a.nbytes, 1) == 0

    def get(self, ptr, shape, dtype=np.float32):
        base, at, n = self.bufs[ptr]
        whole = np.empty(n, np.uint8)
        assert self.rt.hipDeviceSynchronize() == 0
        assert self.rt.hipMemcpy(whole.ctypes.data, base, n, 2) == 0
        size = int(np.prod(shape)) * np.dtype(dtype).itemsize
        assert (whole[:at] == 0xA5).all() and (whole[at + size:] == 0xA5).all(), "bytes outside the buffer changed"
        return whole[at:at + size].view(dtype).reshape(shape)

    def close(self):
        for base, _, _ in self.bufs.values():
            self.rt.hipFree(base)
        self.bufs = {}


def bf16_bits(x):
    """Round to the nearest bf16, ties to even (finite values)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def encode(dtype, x):
    """fp32 values in a type's bits, and the float64 values that they stand for."""
    x = np.asarray(x, np.float32)
    if dtype == W.F32:
        return x, x.astype(np.float64)
    if dtype == W.F16:
        h = x.astype(np.float16)
        return h.view(np.uint16), h.astype(np.float64)
    b = bf16_bits(x)
    return b, decode(W.BF16, b)


def decode(dtype, bits):
    if dtype == W.F32:
        return bits.view(np.float32).astype(np.float64)
    if dtype == W.F16:
        return bits.view(np.float16).astype(np.float64)
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def bits_dtype(dtype):
    return np.float32 if dtype == W.F32 else np.uint16


def mx_quantize(x):
    """(codes [n, cols], scales [n, cols / 32]) of float64 rows."""
    b = np.asarray(x, np.float64).reshape(x.shape[0], -1, 32)
    finite = np.isfinite(b).all(-1)
    b = np.where(finite[..., None], b, 0)
    most = np.abs(b).max(-1)
    e = np.clip(np.frexp(most)[1] - 1 - 2, -127, 127)
    e = np.where(most > 0, e, -127)
    m = np.minimum(np.abs(b) / np.ldexp(1.0, e)[..., None], 6)
    # the nearest grid value; of two equally near the one with an even code
    d = np.abs(m[..., None] - GRID)
    near = d == d.min(-1, keepdims=True)
    first = near.argmax(-1)
    second = 7 - near[..., ::-1].argmax(-1)
    codes = np.where(first % 2 == 0, first, second) | (np.signbit(b) << 3)
    return (np.where(finite[..., None], codes, 0).astype(np.uint8).reshape(x.shape),
            np.where(finite, e + 127, 255).astype(np.uint8))


def mx_values(codes, scales):
    v = GRID[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return (v.reshape(codes.shape[0], -1, 32) * s[..., None]).reshape(codes.shape)


def mx_rows(codes, scales):
    """Codes [n, cols] and scales in the device layout of MXFP4 rows."""
    n, cols = codes.shape
    units = -(-cols // 128)
    c = np.zeros((n, units * 128), np.uint8)
    c[:, :cols] = codes
    s = np.zeros((n, units * 4), np.uint8)
    s[:, :scales.shape[1]] = scales
    c = c[:, ::2] | c[:, 1::2] << 4
    return (np.ascontiguousarray(c.reshape(n, units, 64).transpose(1, 0, 2)),
            np.ascontiguousarray(s.reshape(n, units, 4).transpose(1, 0, 2)))


def random_mx(rng, rows, cols, low=118, high=126):
    return (rng.integers(0, 16, (rows, cols)).astype(np.uint8),
            rng.integers(low, high, (rows, cols // 32)).astype(np.uint8))


def matrices(rng, fmt, count, rows, cols):
    """`count` matrices: raw bytes and float64 values."""
    if fmt == W.MXFP4:
        q = [random_mx(rng, rows, cols) for _ in range(count)]
        return np.concatenate([W.encode_mxfp4(*m) for m in q]), np.stack([mx_values(*m) for m in q])
    bits, v = encode(W.BF16, rng.standard_normal((count, rows, cols)) * 0.02)
    return bits.reshape(-1).view(np.uint8), v


def silu(x):
    with np.errstate(over="ignore"):
        return x / (1 + np.exp(-x))
