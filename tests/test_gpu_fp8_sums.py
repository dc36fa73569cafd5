"""ml_sum_rows: the joined sums of weight and bias gradients."""
import pytest
import torch

from monoloco_amd import fp8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('rows,n', [(1, 1), (2, 5), (31, 40), (257, 33), (1024, 100), (5000, 7), (0, 9), (300, 8191), (300, 8192), (70, 20001)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_sum_rows(cuda_device, hip_lib, rows, n, dtype):
    """In 64 bits, rounded once: `rows` terms of at most 53 bits each add 2^-53 rows of the magnitudes' sum to half a step of the result."""
    g = torch.Generator().manual_seed(rows + n)
    part = torch.randn((rows, n), generator=g) * torch.exp(2 * torch.randn((rows, 1), generator=g))
    if rows > 4:                                # large ones that cancel
        part[1], part[rows - 2] = 30000.0, -30000.0
    out = torch.full((n,), 7.0, dtype=dtype, device=cuda_device)
    dev = part.to(cuda_device)
    assert hip_lib.ml_sum_rows(dev.data_ptr() if rows else None, rows, n, out.data_ptr(), fp8.DTYPES[dtype], torch.cuda.current_stream().cuda_stream) == 0
    want = part.double().sum(0)
    tol = torch.finfo(dtype).eps / 2 * want.abs() + (rows + 1) * 2.0 ** -53 * part.double().abs().sum(0) + 2.0 ** -25 * (dtype == torch.float16)
    assert bool(((out.cpu().double() - want).abs() <= tol * (1 + 2.0 ** -20)).all())
