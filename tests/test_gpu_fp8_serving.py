"""linear without gradients, on the GPU (tests/test_fp8_host.py has what is asked of the library)."""
import pytest
import torch

from monoloco_amd import fp8
from test_gpu_fp8 import TYPES, data

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('m,n,k', [(1, 9, 34), (300, 200, 257), (1000, 512, 1024)])
def test_linear_without_gradients(cuda_device, m, n, k, dtype):
    """The same bits as in training, without the k x (m + n) transposed codes that a backward pass would need."""
    x = data(1, m, k, dtype).to(cuda_device)
    w, b = (torch.nn.Parameter(t.to(cuda_device)) for t in (data(2, n, k, dtype, 0.1), data(3, 1, n, dtype)[0]))
    want = fp8.linear(x.clone().requires_grad_(True), w, b)
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_allocated()
            y = fp8.linear(x, w, b)
            used = torch.cuda.max_memory_allocated() - before
        assert not y.requires_grad and torch.equal(y, want)
        forward, _, _ = fp8._linear_sizes(m, n, k, False, False, False)
        assert used <= forward + y.numel() * y.element_size() + 2 * 512        # (the allocator's granularity)
