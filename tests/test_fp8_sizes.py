"""Sizes at which the entry points' own arithmetic would overflow are refused on the host (no GPU: nothing is launched)."""
import ctypes

import pytest

P = ctypes.c_void_p(4096)     # never dereferenced: every call below is refused


def test_linear_sizes(hip_lib):
    out = (ctypes.c_int64 * 3)(7, 7, 7)
    for m, n, k in ((1 << 40, 1 << 40, 1 << 40), (1 << 32, 1 << 32, 1 << 32), (1 << 24, 16, 1 << 40), (16, 1 << 40, 1 << 24), (1 << 40, 1 << 24, 16), (1 << 41, 1, 1)):
        assert hip_lib.ml_fp8_linear_sizes(m, n, k, 1, 1, 1, out) != 0 and list(out) == [7, 7, 7]
        assert b'ml_fp8_linear_sizes' in hip_lib.ml_ops_last_error()
        for fn, args in ((hip_lib.ml_fp8_linear, (P, 0, k, P, 0, k, None, 0, P, n, m, n, k, 1, 1, P, P, None)),
                         (hip_lib.ml_fp8_linear_backward, (P, 0, n, P, P, 0, P, 0, P, 0, m, n, k, 1, 1, P, None))):
            assert fn(*args) in (1, 4), (m, n, k)
    # what a card can hold: exact sizes (codes of x and w with rows on 16 bytes, a scale byte per 128, on 256 bytes)
    assert hip_lib.ml_fp8_linear_sizes(1 << 20, 1 << 14, 1 << 14, 0, 0, 0, out) == 0 and out[0] == (1 << 34) + (1 << 27) + (1 << 28) + (1 << 14)


@pytest.mark.parametrize('tile', [0, 1])
def test_quantize(hip_lib, tile):
    for m, n in ((1 << 40, 1 << 40), (1 << 39, 1 << 31), (1 << 31, 1 << 40), (1 << 40, 1 << 24)):
        assert hip_lib.ml_fp8_quantize(P, 0, m, n, n, tile, P, n, P, n, None, 0, None, 0, None, None) == 4
        assert b'too large' in hip_lib.ml_ops_last_error()


def test_matmul(hip_lib):
    big = (1 << 63) - 1
    for m, n, k in ((big, 4, 16), (4, big, 16), (1 << 40, 1 << 33, 16), (1 << 40, 1 << 30, 16), (4, 4, big)):
        assert hip_lib.ml_fp8_matmul(P, k, P, big, 0, P, k, P, big, 0, None, 0, P, 0, big, m, n, k, None, 0, None) in (1, 4), (m, n, k)
    for m, n, k in ((4, 4, big), (big, big, big), (1, 1, 1 << 50), (big, 1, 1 << 20)):
        assert hip_lib.ml_fp8_matmul_work(m, n, k, 0) == 0


def test_norm(hip_lib):
    big = (1 << 63) - 1
    for m, n in ((big, 8), (big, 1 << 20), (1 << 40, 1 << 20)):
        assert hip_lib.ml_rms_norm(P, big, None, 0, 0, P, 0, m, n, 1e-6, None, 0, P, big, None, 0, None, 0, None) == 4
    assert hip_lib.ml_rms_norm_backward(P, big, P, big, None, 0, 0, P, 0, 4, big, 1e-6, P, big, P, P, None) == 4
    assert hip_lib.ml_sum_rows(P, 4, big, P, 0, None) == 4
