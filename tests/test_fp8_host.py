"""What monoloco_amd.fp8 asks of the library, without a GPU: the call is recorded instead of made."""
import pytest
import torch

from monoloco_amd import _lib, fp8


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(fp8, '_device_of', lambda name, *tensors: -1)
    monkeypatch.setattr(fp8, '_run', lambda index, fn, *args: made.append((fn, args)))
    return made


@pytest.mark.parametrize('mode', [torch.enable_grad, torch.no_grad, torch.inference_mode])
def test_linear_prepares_gradients_only_where_they_can_come(calls, mode):
    """Without gradients a layer's own parameters (which require them) cost no transposed codes and nothing is kept."""
    w, b = torch.nn.Parameter(torch.zeros(300, 200)), torch.nn.Parameter(torch.zeros(300))
    for x in (torch.zeros(40, 200), torch.zeros(40, 200, requires_grad=True)):
        calls.clear()
        with mode():
            y = fp8.linear(x, w, b)
        (fn, args), = calls
        assert fn is _lib.load().ml_fp8_linear and len(args) == 17
        on = mode is torch.enable_grad
        assert y.requires_grad == on and tuple(map(bool, args[13:15])) == (on and x.requires_grad, on) and (args[16] is not None) == on
