"""The device memory helpers are synchronous: what is enqueued after them finds their memory written."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
SIZE, N = 4 << 30, 8192


def _write_last(F, b, x, w):
    """The last N bytes of b by a kernel on the library's stream; returns them."""
    F.rownorm_dev(x, 1, N // 4, w, 1e-6, b.ptr + SIZE - N)
    F.synchronize()
    return F.DeviceBuffer.download(Tail(b), np.float32, (N // 4,))


class Tail:
    def __init__(self, b):
        self.ptr, self.nbytes = b.ptr + SIZE - N, N


@pytest.mark.parametrize("how", ["fill", "copy"])
def test_done_when_they_return(gpu, how):
    F = gpu
    x = F.DeviceBuffer.from_array(np.random.default_rng(0).standard_normal(N // 4).astype(np.float32))
    w = F.DeviceBuffer.from_array(np.ones(N // 4, np.float32))
    b, other = F.DeviceBuffer(SIZE), F.DeviceBuffer(SIZE if how == "copy" else 16)
    other.fill(9)
    b.fill(0)
    F.synchronize()
    want = _write_last(F, b, x, w)
    assert want.any()
    if how == "fill":
        b.fill(5)
    else:
        assert F.lib().fh3_hip_memcpy_dtod(b.ptr, other.ptr, SIZE) == 0
    assert np.array_equal(_write_last(F, b, x, w), want)
