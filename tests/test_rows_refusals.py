"""What the moves of rows refuse before anything is launched, and the division they use: no GPU needed."""
import ctypes as C

import numpy as np
import pytest
import torch

import diff_gaussian_rasterization as dgr
from gsplat_host import rows

lib = dgr._lib
FAKE = 0x100000                                      # never dereferenced: the checks fail first


def last():
    return lib.gsr_last_error().decode()


def select(tensors=((FAKE, 0, FAKE, 12),), n_rows=10, n_appended=0, n_out=5, index=FAKE, index_bytes=4, count=None):
    words = (C.c_uint64 * max(1, 4 * len(tensors)))(*[w for t in tensors for w in t])
    return lib.gsr_select_rows(len(tensors) if count is None else count, words, n_rows, n_appended, n_out, index, index_bytes, None)


def test_select_checks():
    assert select(count=-1) == -1
    assert lib.gsr_select_rows(2, None, 1, 0, 1, FAKE, 4, None) == -1
    for kw in ({"n_rows": 1 << 31}, {"n_out": 1 << 31}, {"n_rows": 1 << 30, "n_appended": 1 << 30}, {"n_rows": (1 << 64) - 1, "n_appended": 1},
               {"n_rows": 1, "n_appended": (1 << 64) - 1}):
        assert select(**kw) == -1 and "rows" in last(), kw
    for nbytes in (0, 1, 2, 16):
        assert select(index_bytes=nbytes) == -1 and "index of" in last()
    assert select(index=None) == -1 and select(index=FAKE + 2) == -1 and select(index=FAKE + 4, index_bytes=8) == -1
    assert select(tensors=((0, 0, FAKE, 12),)) == -1 and "null pointer in tensor 0" in last()
    assert select(tensors=((FAKE, 0, FAKE, 4), (FAKE, 0, 0, 12))) == -1 and "null pointer in tensor 1" in last()
    assert select(tensors=((FAKE, 0, FAKE, 1 << 31),)) == -1 and "rows of" in last()
    assert select(tensors=((FAKE, 0, FAKE, 1 << 30),), n_out=1 << 10) == -1 and "too large" in last()
    # nothing to do is no error, whatever the pointers
    assert select(n_out=0, index=None) == 0 and select(tensors=(), n_out=5) == 0 and select(tensors=((0, 0, 0, 0),)) == 0


def test_keep_checks():
    nb = lib.gsr_keep_rows_bytes()
    assert nb % 256 == 0
    assert lib.gsr_keep_rows(1 << 31, FAKE, FAKE, FAKE, 1, FAKE, nb, None) == -1 and "rows" in last()
    for hole in range(3):
        ptrs = [FAKE, FAKE, FAKE]
        ptrs[hole] = None
        assert lib.gsr_keep_rows(10, *ptrs, 1, FAKE, nb, None) == -1 and "null" in last()
    assert lib.gsr_keep_rows(10, FAKE, FAKE, FAKE + 4, 1, FAKE, nb, None) == -1 and "aligned" in last()
    assert lib.gsr_keep_rows(10, FAKE, FAKE, FAKE, 1, FAKE, nb - 1, None) == -3
    assert lib.gsr_keep_rows(10, FAKE, FAKE, FAKE, 1, FAKE + 4, nb, None) == -3
    assert lib.gsr_keep_rows(10, FAKE, FAKE, FAKE, 1, None, nb, None) == -3


def test_python_checks():
    a, b = torch.zeros(4, 3), torch.zeros(5, 3)
    index, keep = torch.zeros(2, dtype=torch.int64), torch.ones(4, dtype=torch.bool)
    for fn, arg in ((rows.select_rows, index), (rows.compact_rows, keep)):
        with pytest.raises(ValueError, match="on the GPU"):
            fn([a], arg)
        with pytest.raises(ValueError, match="no tensors"):
            fn([], arg)


def test_the_division_by_multiplication_is_exact():
    """q = (t + ((n - t) >> 1)) >> (l - 1), t = mulhi(m, n), as the kernel forms it, against integer division."""
    rng = np.random.default_rng(0)
    ns = np.unique(np.concatenate([np.arange(70_000), 2 ** 32 - 1 - np.arange(2000), 2 ** 31 + np.arange(-2000, 2000),
                                   rng.integers(0, 2 ** 32, 50_000)])).astype(np.uint64)
    for d in list(range(2, 300)) + [1023, 1024, 1025, 65535, 65536, 65537, 2 ** 31 - 1, 2 ** 30, 2 ** 30 + 1, 1000003]:
        l = max(d - 1, 1).bit_length()
        m = ((((1 << l) - d) << 32) // d + 1) & 0xFFFFFFFF
        t = (np.uint64(m) * ns) >> np.uint64(32)
        q = (t + ((ns - t) >> np.uint64(1))) >> np.uint64(l - 1)
        near = np.concatenate([ns, (ns // np.uint64(d)) * np.uint64(d)])
        assert np.array_equal(q, ns // np.uint64(d)), d
        t = (np.uint64(m) * near) >> np.uint64(32)
        assert np.array_equal((t + ((near - t) >> np.uint64(1))) >> np.uint64(l - 1), near // np.uint64(d)), d
