"""Refusals of the 8-bit residual-block entry points that the host decides before any HIP call, and the host-only parts (no GPU)."""
import ctypes

import pytest
import torch

from monoloco_amd import _lib, fp8
from monoloco_amd.train import AdamW, adamw_step

P = ctypes.c_void_p(4096)     # never dereferenced: every call below is refused, or has nothing to do


def _refused(lib, code, text, fn, *args):
    assert fn(*args) == code
    assert text in lib.ml_ops_last_error().decode(), lib.ml_ops_last_error()


def test_quantize_refusals(hip_lib):
    q = hip_lib.ml_fp8_quantize
    _refused(hip_lib, 1, 'bad type', q, P, 7, 4, 4, 4, 0, P, 16, P, 1, None, 0, None, 0, None, None)
    _refused(hip_lib, 1, 'bad type', q, P, 0, -1, 4, 4, 0, P, 16, P, 1, None, 0, None, 0, None, None)
    _refused(hip_lib, 1, 'null pointer', q, None, 0, 4, 4, 4, 0, P, 16, P, 1, None, 0, None, 0, None, None)
    _refused(hip_lib, 1, 'null pointer', q, P, 0, 4, 4, 4, 0, None, 16, P, 1, None, 0, None, 0, None, None)
    _refused(hip_lib, 1, 'null pointer', q, P, 0, 4, 4, 4, 0, P, 16, None, 1, None, 0, None, 0, None, None)
    _refused(hip_lib, 1, 'null pointer', q, P, 0, 4, 4, 4, 0, P, 16, P, 1, P, 16, None, 1, None, None)
    for ldx, ldq, lds, ldqt, ldst in ((129, 130, 2, 16, 1), (130, 129, 2, 16, 1), (130, 130, 1, 16, 1), (130, 130, 2, 3, 1), (130, 130, 2, 16, 0)):
        _refused(hip_lib, 1, 'row stride', q, P, 0, 4, 130, ldx, 0, P, ldq, P, lds, P, ldqt, P, ldst, None, None)
    _refused(hip_lib, 4, 'too large', q, P, 0, 1 << 41, 4, 4, 0, P, 16, P, 1, None, 0, None, 0, None, None)
    _refused(hip_lib, 4, 'too large', q, P, 0, 1 << 33, 4, 4, 0, P, 16, P, 1, None, 0, None, 0, None, None)
    assert q(None, 0, 0, 4, 4, 0, None, 4, None, 1, None, 0, None, 0, None, None) == 0       # nothing to do


def test_matmul_refusals(hip_lib):
    f = hip_lib.ml_fp8_matmul
    _refused(hip_lib, 1, 'bad type', f, P, 16, P, 1, 0, P, 16, P, 1, 0, None, 0, P, 9, 4, 4, 4, 16, None, 0, None)
    _refused(hip_lib, 1, 'bad type', f, P, 16, P, 1, 0, P, 16, P, 1, 0, P, 5, P, 0, 4, 4, 4, 16, None, 0, None)
    _refused(hip_lib, 1, 'null pointer', f, None, 16, P, 1, 0, P, 16, P, 1, 0, None, 0, P, 0, 4, 4, 4, 16, None, 0, None)
    _refused(hip_lib, 1, 'null pointer', f, P, 16, P, 1, 0, P, 16, P, 1, 0, None, 0, None, 0, 4, 4, 4, 16, None, 0, None)
    for lda, ldsa, ldb, ldsb, ldc in ((129, 2, 130, 2, 4), (130, 1, 130, 2, 4), (130, 2, 129, 2, 4), (130, 2, 130, 1, 4), (130, 2, 130, 2, 3)):
        _refused(hip_lib, 1, 'row stride', f, P, lda, P, ldsa, 0, P, ldb, P, ldsb, 0, None, 0, P, 0, ldc, 4, 4, 130, None, 0, None)
    _refused(hip_lib, 4, 'too large', f, P, 16, P, 1, 0, P, 16, P, 1, 0, None, 0, P, 0, 1 << 30, 1 << 30, 1 << 30, 16, None, 0, None)
    assert f(None, 16, None, 1, 0, None, 16, None, 1, 0, None, 0, None, 0, 4, 0, 4, 16, None, 0, None) == 0


def test_matmul_workspace(hip_lib):
    """Only few tiles with a long k are cut, and the parts stay far below what the operands of such a product take."""
    work = hip_lib.ml_fp8_matmul_work
    assert work(0, 5, 5, 0) == work(5, 0, 5, 0) == work(5, 5, 0, 0) == 0
    for m, n, k in ((1, 4096, 4096), (512, 1024, 1024), (65536, 1024, 1024), (8192, 8192, 8192), (4096, 4096, 16384)):
        assert work(m, n, k, 1) == 0 and work(m, n, k, 0) == 0
    for m, n, k in ((1024, 1024, 65536), (145, 568, 17801), (256, 256, 100000), (9, 1024, 65536)):
        for dt in (0, 1, 2):
            parts, rest = divmod(work(m, n, k, dt), m * n * 4)
            assert rest == 0 and 2 <= parts <= 64 and parts <= k // 1024, (m, n, k, dt, parts)


def test_norm_refusals(hip_lib):
    f, b = hip_lib.ml_rms_norm, hip_lib.ml_rms_norm_backward
    _refused(hip_lib, 1, 'bad types', f, P, 8, None, 0, 3, P, 3, 2, 8, 1e-6, None, 0, P, 8, None, 0, None, 0, None)
    _refused(hip_lib, 1, 'bad types', f, P, 8, None, 0, 1, P, 2, 2, 8, 1e-6, None, 0, P, 8, None, 0, None, 0, None)   # fp16 weight, bf16 rows
    _refused(hip_lib, 1, 'not one of y and q', f, P, 8, None, 0, 0, P, 0, 2, 8, 1e-6, None, 0, P, 8, P, 8, P, 1, None)
    _refused(hip_lib, 1, 'not one of y and q', f, P, 8, None, 0, 0, P, 0, 2, 8, 1e-6, None, 0, None, 8, None, 8, None, 1, None)
    _refused(hip_lib, 1, 'row stride', f, P, 7, None, 0, 0, P, 0, 2, 8, 1e-6, None, 0, P, 8, None, 0, None, 0, None)
    _refused(hip_lib, 1, 'row stride', f, P, 8, P, 7, 0, P, 0, 2, 8, 1e-6, None, 0, P, 8, None, 0, None, 0, None)
    _refused(hip_lib, 1, 'row stride', f, P, 8, None, 0, 0, P, 0, 2, 8, 1e-6, P, 7, P, 8, None, 0, None, 0, None)
    _refused(hip_lib, 4, 'too many', f, P, 8, None, 0, 0, P, 0, 1 << 32, 8, 1e-6, None, 0, P, 8, None, 0, None, 0, None)
    _refused(hip_lib, 1, 'null pointer', b, P, 8, P, 8, None, 0, 0, P, 0, 2, 8, 1e-6, P, 8, None, P, None)
    _refused(hip_lib, 1, 'null pointer', b, P, 8, P, 8, None, 0, 0, P, 0, 2, 8, 1e-6, P, 8, P, None, None)
    _refused(hip_lib, 1, 'row stride', b, P, 8, P, 8, P, 7, 0, P, 0, 2, 8, 1e-6, P, 8, P, P, None)
    assert hip_lib.ml_rms_norm_backward_groups(0, 5) == 0 and hip_lib.ml_rms_norm_backward_groups(1, 5) == 1
    assert 1 <= hip_lib.ml_rms_norm_backward_groups(1 << 40, 1 << 20) <= 4096
    _refused(hip_lib, 1, 'bad type', hip_lib.ml_sum_rows, P, 3, 4, P, 8, None)
    _refused(hip_lib, 1, 'null pointer', hip_lib.ml_sum_rows, None, 3, 4, P, 0, None)


def _adamw(lib, numel=(4, 4), dtype=0, step=1, b1=0.9, b2=0.999, eps=1e-8, null=None, scales=False):
    n = len(numel)
    arr = lambda k: (ctypes.c_void_p * n)(*[None if (k, i) == null else 4096 * (i + 1) for i in range(n)])  # noqa: E731
    return lib.ml_adamw_step(n, (ctypes.c_int64 * n)(*numel), arr(0), arr(1), dtype, arr(2), arr(3), arr(4) if scales else None, step, 1e-3, b1, b2, eps,
                             0.01, 0, None)


def test_adamw_refusals(hip_lib):
    assert _adamw(hip_lib, dtype=4) == 1 and b'bad type' in hip_lib.ml_ops_last_error()
    assert _adamw(hip_lib, step=0) == 1 and b'counted from 1' in hip_lib.ml_ops_last_error()
    for kw in (dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(b1=float('nan'))):
        assert _adamw(hip_lib, **kw) == 1 and b'betas' in hip_lib.ml_ops_last_error()
    for k in range(5):
        assert _adamw(hip_lib, null=(k, 1), scales=True) == 1 and b'tensor 1 has a null pointer' in hip_lib.ml_ops_last_error()
    assert _adamw(hip_lib, numel=(4, -1)) == 4
    assert _adamw(hip_lib, numel=()) == 0


def test_no_cpu_fallback():
    x = torch.zeros(4, 8)
    with pytest.raises(_lib.MonolocoHipError):
        fp8.quantize(x)
    with pytest.raises(_lib.MonolocoHipError):
        fp8.linear(x, torch.zeros(3, 8))
    with pytest.raises(_lib.MonolocoHipError):
        fp8.rms_norm(x, torch.ones(8))
    with pytest.raises(_lib.MonolocoHipError):
        fp8.matmul(x.to(fp8.CODES), torch.ones(4, 1).to(fp8.SCALES), x.to(fp8.CODES), torch.ones(4, 1).to(fp8.SCALES))
    with pytest.raises(_lib.MonolocoHipError):
        adamw_step([x], [x], [x.clone()], [x.clone()], step=1)
    with pytest.raises(_lib.MonolocoHipError):
        p = torch.nn.Parameter(torch.zeros(3))
        p.grad = torch.zeros(3)
        AdamW([p]).step()


def test_adamw_arguments():
    p = torch.zeros(3)
    adamw_step([], [], [], [], step=1)
    with pytest.raises(ValueError, match='counted from 1'):
        adamw_step([p], [p], [p], [p], step=0)
    with pytest.raises(ValueError, match='1 parameters, 0 gradients'):
        adamw_step([p], [], [p], [p], step=1)
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0)):
        with pytest.raises(ValueError):
            AdamW([torch.nn.Parameter(p.clone())], **kw)
