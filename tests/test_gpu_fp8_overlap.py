"""matmul into a buffer that also holds what it reads (tests/test_fp8_overlap.py has the layouts)."""
import pytest
import torch

from monoloco_amd import fp8
from test_gpu_fp8 import operands

pytestmark = pytest.mark.gpu


def test_bias_beside_and_inside_the_result(cuda_device):
    m, n, k = 70, 40, 260
    a = [t.to(cuda_device) for t in operands(1, m, n, k, False, True)]
    bias = torch.arange(float(n), device=cuda_device)
    want = fp8.matmul(*a, bias=bias, out_dtype=torch.float32)
    big = torch.zeros((m + 1, 2 * n), device=cuda_device)
    for v in (big[0, n:], big[m - 1, n:], big[m, :n], big[m, 3:n + 3]):       # between the rows, behind them
        big.zero_()
        v.copy_(bias)
        assert torch.equal(fp8.matmul(*a, bias=v, out=big[:m, :n]), want) and torch.equal(v, bias)
    for v in (big[0, :n], big[m - 1, :n], big[5, 1:n + 1], big[5, n - 1:2 * n - 1], big.view(-1)[2 * n - 1:3 * n - 1]):
        big.zero_()
        v.copy_(bias)
        before = big.clone()
        with pytest.raises(ValueError, match='shares memory with bias'):
            fp8.matmul(*a, bias=v, out=big[:m, :n])
        assert torch.equal(big, before)
