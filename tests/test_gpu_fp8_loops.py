"""Loops that only large calls take more than once (bounds: tests/test_gpu_fp8.py; the 64-bit forms on the GPU)."""
import pytest
import torch

import ref8 as R
import test_gpu_fp8
from monoloco_amd import fp8
from test_gpu_fp8 import U, data, half

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('m,n', [(8300, 1024), (4101, 2048), (2100, 2050), (1100, 8200), (1030, 16390), (513, 16384)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_norm_backward_of_more_rows_than_workgroups(cuda_device, m, n, dtype):
    """Every workgroup takes several rows: the reduction's shared memory is used again, the weight's sums go on, the next row is fetched ahead."""
    x, dy, dh = (data(s, m, n, dtype, 0.3).to(cuda_device) for s in (1, 2, 3))
    w = (1 + 0.2 * data(4, 1, n, torch.float32)[0]).to(dtype).to(cuda_device)
    r = torch.zeros_like(x)
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
    y, h = fp8.rms_norm(leaves[0], leaves[2], residual=leaves[1])
    assert torch.equal(h, x)
    got = [torch.autograd.grad((y, h), leaves, (dy, dh), retain_graph=True) for _ in range(2)]
    assert all(torch.equal(s, t) for s, t in zip(*got))
    dx, dr, dw = got[0]
    ex, ew, ax, aw = R.rms_norm_backward(dy, x, w, dh, 1e-6)
    c, sub = 70 + n / 1024, 2.0 ** -25 if dtype == torch.float16 else 0
    assert torch.equal(dx, dr)
    assert bool(((dx.double() - ex).abs() <= 3 * c * U * ax + half(dtype) * ex.abs() + sub).all())
    assert bool(((dw.double() - ew).abs() <= (m + c) * U * aw + half(dtype) * ew.abs() + sub).all())
    wy, _ = R.rms_norm(x, w, None, 1e-6)
    assert bool(((y.detach().double() - wy).abs() <= (c * U + half(dtype)) * wy.abs() + sub).all())


@pytest.mark.parametrize('m,n,k', [(6000, 6152, 1152), (4100, 9000, 2048)])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_matmul_three_tiles_a_workgroup(cuda_device, m, n, k, dtype):
    """More than 512 tiles of 256 x 256: the bias's two places and the ring's slots come round."""
    test_gpu_fp8.test_matmul_many_tiles(cuda_device, m, n, k, True, dtype)
