"""O_DIRECT requests whose buffer the kernel cannot pin (memory without pages of its own, as a GPU driver may map pinned
memory): the data arrive all the same, and an address that is none stays an error."""
import ctypes
import mmap
import os

import numpy as np
import pytest

import bofhip

SIZE = 1 << 16


@pytest.fixture
def unpinnable():
    """memory of memfd_secret: the kernel copies to and from it and refuses to pin it"""
    fd = ctypes.CDLL(None, use_errno=True).syscall(447, 0)
    if fd < 0:
        pytest.skip("the kernel has no memfd_secret")
    os.ftruncate(fd, SIZE)
    m = mmap.mmap(fd, SIZE)
    view = np.frombuffer(m, np.uint8)
    yield view
    os.close(fd)


@pytest.mark.parametrize("use_aio", [0, 1])
@pytest.mark.parametrize("stride,n,length", [(0, 1, SIZE), (8192, 4, 4096)])
def test_direct_io_into_memory_that_cannot_be_pinned(tmp_path, unpinnable, use_aio, stride, n, length):
    path = str(tmp_path / "data")
    data = np.random.default_rng(1).integers(0, 256, SIZE, np.uint8)
    data.tofile(path)
    fd = os.open(path, os.O_RDWR | os.O_DIRECT)
    try:
        with pytest.raises(OSError):   # (what the test is about holds here)
            os.preadv(fd, [unpinnable], 0)
        L = bofhip.lib()
        at = unpinnable.ctypes.data
        assert L.bof_file_sread(fd, 0, stride, n, length, at, use_aio) == 0
        rows = data.reshape(-1, stride or SIZE)[:n, :length]
        assert np.array_equal(unpinnable[:n * length].reshape(n, length), rows)
        unpinnable[:n * length] ^= 0xFF
        assert L.bof_file_swrite(fd, 0, stride, n, length, at, use_aio) == 0
        want = data.copy().reshape(-1, stride or SIZE)
        want[:n, :length] ^= 0xFF
        assert np.array_equal(np.fromfile(path, np.uint8), want.reshape(-1))
        assert L.bof_file_sread(fd, 0, 0, 1, 4096, 1 << 12, use_aio) != 0   # nothing is mapped there
        assert b"Bad address" in L.bof_last_error()
    finally:
        L.bof_file_forget(fd)
        os.close(fd)
