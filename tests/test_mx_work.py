"""The workspace a microscaled product asks for (no GPU: nothing is launched)."""

import pytest

from tensorfold_b200 import _lib


@pytest.mark.parametrize("n,k,most", [(17408, 5120, 4), (5120, 17408, 4), (6144, 5120, 8), (1024, 5120, 16), (4096, 4096, 16), (128, 100000, 0)])
def test_windows_may_need_work(n, k, most):
    """Up to ``most`` rows (segments of 1024 inputs in a K slice, 24 of them over all rows) a block quantises its rows itself.  Beyond that a
    call without work, or with a byte less, is refused, at window sizes too."""

    lib = _lib.lib()
    x, w, out, work = 0x10000, 0x20000, 0x30000, 0x40000
    for m in range(1, 17):
        need = lib.tf_mx_matmul_bytes(m, n, k)
        assert (need == 0) == (m <= most), m
        if need:
            for area, size in ((None, 0), (None, need), (work, need - 1)):
                assert lib.tf_mx_matmul(x, k, m, w, n, k, out, n, 0, 0, 0.0, area, size, 0, None) == -1, m
                assert b"tf_mx_matmul_bytes" in lib.tf_last_error()
