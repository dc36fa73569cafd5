"""ml_fp8_matmul's result may not lie on what the call reads: decided on the host (no GPU: every call here is refused)."""
import ctypes

import numpy as np


def product(lib, m=5, n=6, k=130, a=(1 << 20, 144), sa=(2 << 20, 2), b=(3 << 20, 144), sb=(4 << 20, 2), bias=5 << 20, c=(6 << 20, 6), dtype=0):
    p = lambda x: ctypes.c_void_p(int(x))  # noqa: E731
    return lib.ml_fp8_matmul(p(a[0]), a[1], p(sa[0]), sa[1], 0, p(b[0]), b[1], p(sb[0]), sb[1], 0, p(bias), 0, p(c[0]), dtype, c[1], m, n, k, None, 0, None)


def test_refused(hip_lib):
    for kw in (dict(bias=(6 << 20) + 5 * 24 - 4), dict(bias=(6 << 20) - 20), dict(c=(5 << 20, 6)), dict(c=(1 << 20, 6)), dict(c=((3 << 20) + 5 * 144 + 129, 6)),
               dict(c=((2 << 20) + 9, 6)), dict(c=((4 << 20) - 5 * 24 + 1, 6)), dict(c=(6 << 20, 100), bias=(6 << 20) + 3 * 400 + 20), dict(c=(6 << 20, 36), a=((6 << 20) + 20, 144))):
        assert product(hip_lib, **kw) == 1 and b'shares memory' in hip_lib.ml_ops_last_error(), kw


def test_against_every_byte(hip_lib):
    """Which layouts are refused, against the sets of bytes: bias and codes inside and between the rows of a strided result.  (Layouts that are
    apart are not passed to the entry point, which would launch: the decision itself is what ml_debug_areas_apart returns.)"""
    rng = np.random.default_rng(1)
    seen = [0, 0]
    for _ in range(3000):
        rows, width = rng.integers(1, 6, 2), rng.integers(1, 9, 2)
        pitch = width + rng.integers(0, 12, 2)
        if rng.random() < 0.3:
            pitch[1] = pitch[0] = max(pitch)
        at = 1000 + rng.integers(0, 60, 2)
        touched = [{int(at[i] + r * pitch[i] + x) for r in range(rows[i]) for x in range(width[i])} for i in range(2)]
        apart = not touched[0] & touched[1]
        args = [int(v) for i in range(2) for v in (at[i], pitch[i], width[i], rows[i])]
        got = bool(hip_lib.ml_debug_areas_apart(*args))
        if rows[1] == 1 or pitch[0] == pitch[1]:
            assert got == apart or (got is False and rows[1] > 1), args      # (equal pitches: bands; the same band at other rows is refused)
        assert apart or not got, args                                        # nothing that overlaps passes
        seen[got] += 1
    assert min(seen) > 300, seen
