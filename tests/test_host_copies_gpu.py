"""Copies from the host that are said to be done when the call returns."""
import ctypes as C

import numpy as np
import pytest

from _support import load_package

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nbytes", [4096, 81920, 184320, 3000001])
def test_what_follows_a_blocking_copy_sees_it_on_any_stream(nbytes):
    """From pageable memory; the stream behind it is one that does not wait for the default stream."""
    g = load_package().ffi
    g.require_device()
    lib, stream = g.cuda(), C.c_void_p()
    g.check(lib.greta_cuda_stream_create(C.byref(stream)))
    a, b, rounds = g.DeviceBuffer(nbytes, zero=True), g.DeviceBuffer(nbytes, zero=True), 400 if nbytes < 1 << 20 else 60
    src = [np.full(nbytes, i, np.uint8) for i in range(7)]
    late = 0
    for i in range(rounds):
        g.check(lib.greta_cuda_memcpy_h2d_sync(a.ptr, src[i % 7].ctypes.data, nbytes))
        g.check(lib.greta_cuda_memcpy_d2d(b.ptr, a.ptr, nbytes, stream))
        g.check(lib.greta_cuda_stream_synchronize(stream))
        late += not np.array_equal(b.download(np.uint8), src[i % 7])
    lib.greta_cuda_stream_destroy(stream)
    assert late == 0
