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


def test_matmul_refuses_operands_with_a_history(calls):
    """Codes cast from what needs a gradient would lose it without a word."""
    x, w = torch.zeros(4, 128, requires_grad=True), torch.zeros(5, 128)
    s = torch.ones(4, 1, requires_grad=True)
    for kw in (dict(a=x.to(fp8.CODES)), dict(b=torch.zeros(5, 128, requires_grad=True).to(fp8.CODES)), dict(a_scale=s.to(fp8.SCALES)),
               dict(b_scale=torch.ones(5, 1, requires_grad=True).to(fp8.SCALES)), dict(bias=torch.zeros(5, requires_grad=True))):
        args = dict(a=x.detach().to(fp8.CODES), a_scale=s.detach().to(fp8.SCALES), b=w.to(fp8.CODES), b_scale=torch.ones(5, 1).to(fp8.SCALES))
        args.update(kw)
        assert args[next(iter(kw))].requires_grad
        with pytest.raises(ValueError, match='not differentiable'):
            fp8.matmul(**args)
        assert not calls
        with torch.no_grad():
            assert fp8.matmul(**args).shape == (4, 5)
        assert len(calls) == 1
        calls.clear()
