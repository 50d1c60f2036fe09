"""dropout at the sizes that its numbers of rows and of columns allow."""
import ctypes
import gc

import numpy as np
import pytest

from tests import blocks_reference as R
from tests.test_blocks_host import BF16, F32, S, lib


def test_sizes_that_are_refused():
    """Rows, and rows times groups of eight columns, of 2^32 and more: refused before anything is launched."""
    L = lib()
    L.musapy_kernels_take_error()
    for shape in ((1 << 32, 8), (1 << 31, 2, 1), (1 << 31, 16), (1, (1 << 35) - 7), ((1 << 35) - 7,), (1 << 40,), (2, 1 << 34),
                  (1 << 16, 1 << 16, 1), (1 << 32, 1 << 32, 8), (1 << 63, 2, 8)):
        n = len(shape)
        st = (ctypes.c_ssize_t * n)(*[0] * (n - 1), 1)
        for dtype in (F32, BF16):
            assert L.musapy_dropout_v1(64, 64, dtype, n, (S * n)(*shape), st, 1, 1, 0, None) == -1, shape
            assert L.musapy_kernels_take_error() == 6, shape
    for shape in ((1 << 32, 0), (0, 1 << 40), (1 << 63, 2, 0)):
        n = len(shape)
        st = (ctypes.c_ssize_t * n)(*[0] * (n - 1), 1)
        assert L.musapy_dropout_v1(None, None, F32, n, (S * n)(*shape), st, 1, 1, 0, None) == 0, shape


@pytest.mark.gpu
def test_more_than_2_32_columns():
    """One row of 2^32 + 11 columns (about 17 GB with its result), at places on both sides of the 32-bit numbers."""
    import musapy_amd as ms

    n, p, seed, offset = (1 << 32) + 11, 0.4, 2 ** 33 + 5, 6
    x = np.full(n, 0x3F80, np.uint16)  # 1.0
    X = ms.array(x, dtype="bf16")
    del x
    Y = ms.dropout(X, p, seed=seed, offset=offset)
    kept = float(R.rounded(np.array([np.float32(R.keep_scale(p))]), "bf16")[0])
    m = 0xFFFFFFFF
    for at in (0, (1 << 31) - 16, 1 << 31, (1 << 32) - 16, (1 << 32) - 8, 1 << 32, (1 << 32) + 8):
        words = R.philox4x32((at // 8, 0, offset & m, offset >> 32), (seed & m, seed >> 32))
        keep = [h >= round(p * 65536) for w in words for h in (w & 0xFFFF, w >> 16)]
        got = R.values(Y[at:min(at + 8, n)])
        assert got.tolist() == [kept if k else 0.0 for k in keep][:len(got)], at
    del X, Y
    gc.collect()
    ms.synchronize()
    ms.empty_cache()
