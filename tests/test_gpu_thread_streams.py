"""Products on hipStreamPerThread whose scratch other streams share: such a call returns while its work runs, and other
streams' calls come after it, also when its thread has ended."""
import ctypes as C
import threading

import numpy as np
import pytest

from experts_fixture import Device, encode
from tinyoai_amd import weights as W

pytestmark = pytest.mark.gpu

PER_THREAD = 2  # hipStreamPerThread
ROWS, COLS, N = 900, 1536, 70


class Products:
    """A weight, its products' inputs and results, and work of tens of milliseconds to put in front of a call."""

    def __init__(self, shared):
        from tinyoai_amd import hip
        self.hip, self.dev = hip, Device()
        self.rt = rt = self.dev.rt
        rng = np.random.default_rng(61)
        bits = encode(W.F16, rng.standard_normal((ROWS, COLS)))[0]
        self.w = hip.Weight(W.Tensor(W.F16, ROWS, COLS, bits.reshape(-1).view(np.uint8)))
        self.x = [self.dev.put(rng.standard_normal((N, COLS)).astype(np.float32)) for _ in range(2)]
        self.y = [self.dev.put(np.zeros((N, ROWS), np.float32)) for _ in range(2)]
        self.want = []
        for x, y in zip(self.x, self.y):
            self.w.mul_device(x, N, y)
            self.want.append(self.dev.get(y, (N, ROWS)).copy())
            self.dev.fill(y, np.full((N, ROWS), np.nan, np.float32))
        self.streams = [C.c_void_p() for _ in range(10)]
        for st in self.streams:
            assert rt.hipStreamCreateWithFlags(C.byref(st), 1) == 0
        self.call = self.w.mul_device if shared else self.w.mul_device_noalloc
        z = self.dev.put(np.zeros((N, ROWS), np.float32))
        for st in self.streams[:8]:  # all of the weight's buffers taken: the next streams share one
            self.call(self.x[0], N, z, st.value)
        self.rows, self.out = (self.dev.room(8192 * 4096 * 4) for _ in range(2))
        self.offsets = self.dev.put(np.array([0, 8192], np.int32))
        assert rt.hipDeviceSynchronize() == 0

    def long(self, stream):
        for _ in range(6):
            self.hip.attention(W.F32, self.rows, 4096, 32, self.rows, 4096, self.rows, 4096, 32, 128, 0.1, False, self.offsets,
                               self.offsets, 1, 8192, 8192, self.out, 4096, stream)

    def read(self, i):
        """y[i] as it is, without waiting for any other stream."""
        got = np.empty((N, ROWS), np.float32)
        st = self.streams[9]
        assert self.rt.hipMemcpyAsync(C.c_void_p(got.ctypes.data), C.c_void_p(self.y[i]), C.c_size_t(got.nbytes), 2, st) == 0
        assert self.rt.hipStreamSynchronize(st) == 0
        return got

    def thread(self, work):
        errors = []

        def run():
            try:
                assert self.rt.hipSetDevice(0) == 0
                work()
            except BaseException as e:  # noqa: BLE001
                errors.append(e)

        t = threading.Thread(target=run)
        t.start()
        t.join()
        if errors:
            raise errors[0]

    def close(self):
        self.rt.hipDeviceSynchronize()
        for st in self.streams:
            self.rt.hipStreamDestroy(st)
        self.w.close()
        self.dev.close()


@pytest.fixture(params=[True, False], ids=["shared", "library"])
def products(request):
    p = Products(request.param)
    yield p
    p.close()


def test_thread_stream_calls_do_not_wait(products):
    p = products
    states = []

    def work():
        p.long(PER_THREAD)
        p.call(p.x[0], N, p.y[0], PER_THREAD)
        states.append(p.rt.hipStreamQuery(C.c_void_p(PER_THREAD)))
        assert p.rt.hipStreamSynchronize(C.c_void_p(PER_THREAD)) == 0

    p.thread(work)
    assert states == [600]  # hipErrorNotReady
    assert np.array_equal(p.read(0), p.want[0])


def test_calls_come_after_those_of_ended_threads(products):
    """The thread's work runs for some 50 ms when it ends; the next stream's call ends after it."""
    p = products

    def work():
        p.long(PER_THREAD)
        p.call(p.x[0], N, p.y[0], PER_THREAD)

    for _ in range(2):
        p.thread(work)
        p.call(p.x[1], N, p.y[1], p.streams[8].value)
        assert p.rt.hipStreamSynchronize(p.streams[8]) == 0
        assert np.array_equal(p.read(0), p.want[0]) and np.array_equal(p.read(1), p.want[1])
        for y in p.y:
            p.dev.fill(y, np.full((N, ROWS), np.nan, np.float32))
