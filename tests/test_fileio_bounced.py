"""O_DIRECT requests whose buffer the kernel cannot pin stay O_DIRECT: they are counted, leave no pages in the page cache, neither clean
nor waiting to be written, and an address that is none ends in an error."""
import ctypes
import mmap
import os
import subprocess
import sys

import numpy as np
import pytest

import bofhip
from test_fileio_unpinnable import SIZE, unpinnable  # noqa: F401 (a fixture)

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture
def direct_file(tmp_path):
    path = str(tmp_path / "data")
    np.random.default_rng(1).integers(0, 256, 4 * SIZE, np.uint8).tofile(path)
    fd = os.open(path, os.O_RDWR | os.O_DIRECT)
    os.fsync(fd)
    yield fd, path
    bofhip.lib().bof_file_forget(fd)
    os.close(fd)


def moved(call):
    before = bofhip.file_bounced_bytes()
    assert call() == 0
    return tuple(b - a for a, b in zip(before, bofhip.file_bounced_bytes()))


@pytest.mark.parametrize("use_aio", [0, 1])
@pytest.mark.parametrize("stride,n,length", [(0, 1, SIZE), (8192, 8, 4096)])
def test_they_are_counted(direct_file, unpinnable, use_aio, stride, n, length):  # noqa: F811
    L, (fd, _), at = bofhip.lib(), direct_file, unpinnable.ctypes.data
    assert moved(lambda: L.bof_file_sread(fd, 0, stride, n, length, at, use_aio)) == (n * length, 0)
    assert moved(lambda: L.bof_file_swrite(fd, 0, stride, n, length, at, use_aio)) == (0, n * length)
    own = mmap.mmap(-1, SIZE)                                   # memory that can be
    at = ctypes.addressof(ctypes.c_char.from_buffer(own))
    assert moved(lambda: L.bof_file_sread(fd, 0, stride, n, length, at, use_aio)) == (0, 0)
    assert moved(lambda: L.bof_file_swrite(fd, 0, stride, n, length, at, use_aio)) == (0, 0)


class CacheStat(ctypes.Structure):
    _fields_ = [(f, ctypes.c_uint64) for f in ("cached", "dirty", "writeback", "evicted", "recently_evicted")]


def pages(path):
    """CacheStat of a file, or None where the kernel does not say (cachestat, Linux 6.5)"""
    fd = os.open(path, os.O_RDONLY)
    try:
        st, span = CacheStat(), (ctypes.c_uint64 * 2)(0, 0)
        return st if ctypes.CDLL(None, use_errno=True).syscall(451, fd, span, ctypes.byref(st), 0) == 0 else None
    finally:
        os.close(fd)


@pytest.mark.parametrize("use_aio", [0, 1])
@pytest.mark.parametrize("stride,n,length", [(0, 1, SIZE), (8192, 8, 4096)])
def test_they_pass_the_page_cache_by(direct_file, unpinnable, use_aio, stride, n, length):  # noqa: F811
    L, (fd, path) = bofhip.lib(), direct_file
    os.posix_fadvise(fd, 0, 0, os.POSIX_FADV_DONTNEED)
    before = pages(path)
    if before is None or before.cached:
        pytest.skip("the kernel does not say what of this file system is cached, or keeps it")
    assert moved(lambda: L.bof_file_sread(fd, 0, stride, n, length, unpinnable.ctypes.data, use_aio)) == (n * length, 0)
    assert pages(path).cached == 0
    unpinnable[:] = 7
    assert moved(lambda: L.bof_file_swrite(fd, 0, stride, n, length, unpinnable.ctypes.data, use_aio)) == (0, n * length)
    after = pages(path)
    assert (after.cached, after.dirty, after.writeback) == (0, 0, 0)


PIECES = """
import ctypes, mmap, os, sys
import numpy as np
import bofhip
L, path, total = bofhip.lib(), sys.argv[1], 6 << 20
stride, n, length = {stride}, {n}, {length}
secret = ctypes.CDLL(None, use_errno=True).syscall(447, 0)     # memfd_secret
if secret < 0:
    sys.exit(print("skip: no memfd_secret"))
os.ftruncate(secret, n * length)
try:
    buf = np.frombuffer(mmap.mmap(secret, n * length), np.uint8)
    buf[:] = 0
except OSError:
    sys.exit(print("skip: no room for secret memory"))
data = np.random.default_rng(2).integers(0, 256, total, np.uint8)
data.tofile(path)
fd = os.open(path, os.O_RDWR | os.O_DIRECT)
for use_aio in (0, 1):     # (large writes without it may be stores through a mapping: counted with it)
    before = bofhip.file_bounced_bytes()
    starts = [4096 + s * stride for s in range(n)]
    buf[:] = 0
    assert L.bof_file_sread(fd, 4096, stride, n, length, buf.ctypes.data, use_aio) == 0, L.bof_last_error()
    assert np.array_equal(buf, np.concatenate([data[s:s + length] for s in starts]))
    buf ^= 0xA5
    assert L.bof_file_swrite(fd, 4096, stride, n, length, buf.ctypes.data, use_aio) == 0, L.bof_last_error()
    for i, s in enumerate(starts):
        data[s:s + length] = buf[i * length:(i + 1) * length]
    assert np.array_equal(np.fromfile(path, np.uint8), data)
assert bofhip.file_bounced_bytes() == (before[0] + n * length, before[1] + n * length)
L.bof_flash_release()
assert L.bof_file_sread(fd, 4096, stride, n, length, buf.ctypes.data, 1) == 0
print("whole")
"""


@pytest.mark.parametrize("stride,n,length", [(0, 1, 5 << 20), (2560 << 10, 2, 2304 << 10), (8192, 500, 4096), (0, 1, 20480), (3 << 20, 2, 1 << 20)])
@pytest.mark.parametrize("engine", ["aio", "uring"])
def test_they_arrive_whole_in_pieces(tmp_path, engine, stride, n, length):
    """Requests below, between and above what is copied at a time (BOF_BOUNCE_KIB: here 1 MiB)."""
    code = PIECES.replace("{stride}", str(stride)).replace("{n}", str(n)).replace("{length}", str(length))
    r = subprocess.run([sys.executable, "-c", code, str(tmp_path / "data")], cwd=HERE, capture_output=True, text=True, timeout=120,
                       env=dict(os.environ, BOF_BOUNCE_KIB="1024", BOF_IO_ENGINE=engine, PYTHONPATH=os.pathsep.join(sys.path)))
    if "skip" in r.stdout:
        pytest.skip(r.stdout)
    assert r.returncode == 0 and "whole" in r.stdout, (r.returncode, r.stdout, r.stderr)


FORKED = """
import ctypes, mmap, os, sys
import numpy as np
import bofhip
L, path, size = bofhip.lib(), sys.argv[1], 1 << 20
secret = ctypes.CDLL(None, use_errno=True).syscall(447, 0)     # memfd_secret
if secret < 0:
    sys.exit(print("skip: no memfd_secret"))
os.ftruncate(secret, 2 * size)
try:
    buf = np.frombuffer(mmap.mmap(secret, 2 * size), np.uint8)
    buf[:] = 0
except OSError:
    sys.exit(print("skip: no room for secret memory"))
data = np.random.default_rng(2).integers(0, 256, 2 * size, np.uint8)
data.tofile(path)
fd = os.open(path, os.O_RDWR | os.O_DIRECT)
def read(part):
    mine = buf[part * size:(part + 1) * size]
    mine[:] = 0
    assert L.bof_file_sread(fd, part * size, 0, 1, size, mine.ctypes.data, 0) == 0, L.bof_last_error()
    return np.array_equal(mine, data[part * size:(part + 1) * size])
assert read(0) and bofhip.file_bounced_bytes()[0] == size
child = os.fork()
good = all([read(child == 0) for _ in range(200)])
if child == 0:
    os._exit(0 if good else 1)
assert os.waitstatus_to_exitcode(os.waitpid(child, 0)[1]) == 0 and good
print("apart")
"""


def test_a_forked_process_has_its_own(tmp_path):
    """Parent and child read at once what each of them has to copy: neither finds the other's bytes."""
    r = subprocess.run([sys.executable, "-c", FORKED, str(tmp_path / "data")], cwd=HERE, capture_output=True, text=True, timeout=120,
                       env=dict(os.environ, PYTHONPATH=os.pathsep.join(sys.path)))
    if "skip" in r.stdout:
        pytest.skip(r.stdout)
    assert r.returncode == 0 and "apart" in r.stdout, (r.returncode, r.stdout, r.stderr)


BAD_WRITE = """
import os, sys
import bofhip
L, path, size = bofhip.lib(), sys.argv[1], 2 << 20
with open(path, "wb") as f:
    f.write(bytes(size))                        # resident pages, without holes
    os.fsync(f.fileno())
fd = os.open(path, os.O_RDWR | os.O_DIRECT)
assert L.bof_file_swrite(fd, 0, 0, 1, size, 1 << 12, 1) != 0                # nothing is mapped there
assert b"Bad address" in L.bof_last_error(), L.bof_last_error()
print("refused")
"""


def test_a_large_write_from_nowhere_is_an_error(tmp_path):
    """(Its pages are resident when it begins, as for the stores through a mapping that a buffered write of this size may use.)"""
    r = subprocess.run([sys.executable, "-c", BAD_WRITE, str(tmp_path / "data")], cwd=HERE, capture_output=True, text=True, timeout=120,
                       env=dict(os.environ, PYTHONPATH=os.pathsep.join(sys.path)))
    assert r.returncode == 0 and "refused" in r.stdout, (r.returncode, r.stdout, r.stderr)
