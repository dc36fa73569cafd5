"""The product with operands of a single row: what a caller gives as its row stride changes nothing (bounds: tests/test_gpu_fp8.py)."""
import pytest
import torch

from monoloco_amd import fp8
from test_gpu_fp8 import F8, TYPES, check_product, operands

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('m,n,k', [(1, 5, 40001), (600, 1, 17801), (1, 300, 20001), (1, 1, 9001), (1, 40, 1111)])
def test_matmul_one_row(cuda_device, hip_lib, m, n, k, dtype):
    a, sa, b, sb = operands(m + n, m, n, k, False, False)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(1))
    dev, bv = [t.to(cuda_device) for t in (a, sa, b, sb)], bias.to(cuda_device)
    pad = k + -k % 16
    wide = [torch.full((t.shape[0], pad), 0x7f, dtype=torch.uint8, device=cuda_device) for t in (a, b)]
    for t, v in zip(wide, (dev[0], dev[2])):
        t[:, :k] = v.view(torch.uint8)
    x, w = (t[:, :k].view(F8) for t in wide)
    c = fp8.matmul(x, dev[1], w, dev[3], bias=bv, out_dtype=dtype)
    check_product(c, a, sa, False, b, sb, False, bias, dtype)
    size = hip_lib.ml_fp8_matmul_work(m, n, k, fp8.DTYPES[dtype])
    work = torch.empty((max(size, 1),), dtype=torch.uint8, device=cuda_device)
    out = torch.empty((m, n), dtype=dtype, device=cuda_device)
    for lda, ldb in ((pad, pad), (pad if m > 1 else k, pad if n > 1 else k), (pad if m > 1 else k + 5, pad if n > 1 else 1 << 40)):
        out.fill_(7)
        assert hip_lib.ml_fp8_matmul(x.data_ptr(), lda, dev[1].data_ptr(), dev[1].stride(0), 0, w.data_ptr(), ldb, dev[3].data_ptr(), dev[3].stride(0), 0, bv.data_ptr(),
                                     fp8.DTYPES[bv.dtype], out.data_ptr(), fp8.DTYPES[dtype], n, m, n, k, work.data_ptr() if size else None, size,
                                     torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(out, c), (lda, ldb)
    # a start that is not on 16 bytes: the plain kernels
    odd = torch.zeros(pad + 16, dtype=torch.uint8, device=cuda_device)[3:3 + k]
    which = 0 if m == 1 else 1
    odd.copy_((x, w)[which].view(torch.uint8)[0])
    odd = odd.view(F8).view(1, k)
    check_product(fp8.matmul(odd if which == 0 else x, dev[1], odd if which == 1 else w, dev[3], bias=bv, out_dtype=dtype), a, sa, False, b, sb, False, bias, dtype)
