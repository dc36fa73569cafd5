"""AdamW's 8-bit moments over groups and gaps, on the GPU (tests/test_adamw_state.py has the numbering itself)."""
import pytest
import torch

import ref8 as R
from monoloco_amd.train import AdamW

pytestmark = pytest.mark.gpu


def codes(o, p):
    return [o.state[p][k].view(torch.uint8).clone() for k in ('exp_avg', 'exp_avg_sq')]


def test_groups_and_types_round_apart(cuda_device):
    """Equal tensors with equal gradients in two groups: the same scales and parameters, other codes (of 4096 roundings, most of them between two
    codes, all falling alike has a chance below 2^-1000)."""
    g = 0.01 * torch.randn(4096, generator=torch.Generator().manual_seed(1)).to(cuda_device)
    a, b = (torch.nn.Parameter(torch.ones(4096, device=cuda_device)) for _ in range(2))
    o = AdamW([{'params': [a]}, {'params': [b]}], lr=1e-2, state_bits=8, seed=3)
    a.grad, b.grad = g.clone(), g.clone()
    o.step()
    assert torch.equal(a, b) and torch.equal(o.state[a]['scales'].view(torch.uint8), o.state[b]['scales'].view(torch.uint8))
    for x, y in zip(codes(o, a), codes(o, b)):
        assert not torch.equal(x, y)


def test_a_missing_gradient_moves_no_other_tensor(cuda_device):
    """The second and fourth of five tensors step as numbers 1 and 3, with or without the others' gradients, and in the library's numbering."""
    shapes = [(7,), (129,), (64,), (1000,), (5,)]
    gen = torch.Generator().manual_seed(2)
    start, grads = [0.1 * torch.randn(s, generator=gen) for s in shapes], [0.01 * torch.randn(s, generator=gen) for s in shapes]
    got = []
    for have in (range(5), (1, 3)):
        ps = [torch.nn.Parameter(t.to(cuda_device)) for t in start]
        o = AdamW(ps, lr=1e-2, state_bits=8, seed=9)
        for i in have:
            ps[i].grad = grads[i].to(cuda_device)
        o.step()
        for i in set(range(5)) - set(have):
            assert torch.equal(ps[i].cpu(), start[i]) and not o.state[ps[i]]
        got.append([codes(o, ps[i]) + [ps[i].detach(), o.state[ps[i]]['scales'].view(torch.uint8)] for i in (1, 3)])
        for i in (1, 3):
            want, _ = R.stochastic(grads[i].double() * (1 - 0.9), R.bits(9, 1, i, grads[i].numel()) & 0xffff, False)
            off = (o.state[ps[i]]['exp_avg'].cpu().float().double() - want).abs()
            assert float((off > 0).double().mean()) <= 0.01 and bool((off <= 1.001 * R.step_of(want)).all())    # (2^-16 of a step: see test_gpu_adamw.py)
    for x, y in zip(*got):
        assert all(torch.equal(s, t) for s, t in zip(x, y))


def test_neighbours_and_shared_gradients(cuda_device):
    """Tensors that touch without a byte between them, one gradient for two of them, a gradient that is its own parameter: allowed.  What shares
    memory is refused and nothing is written."""
    from monoloco_amd.train import adamw_step
    flat, m, v = torch.ones(300, device=cuda_device), torch.zeros(300, device=cuda_device), torch.zeros(300, device=cuda_device)
    g = torch.full((100,), 0.5, device=cuda_device)

    def cut(t, at=(0, 100, 200)):
        return [t[i:i + 100] for i in at]

    def step(ps, gs):
        adamw_step(ps, gs, cut(m), cut(v), step=1, lr=0.1, weight_decay=0.0)

    # the first step moves by lr * sign(g), but for eps (1e-8 / 0.5) and roundings (20 u of 0.1)
    step(cut(flat), [g, flat[100:200], g])
    assert bool(((flat - 0.9).abs() <= 0.1 * (2e-8 + 20 * 2.0 ** -24) + 2 * 2.0 ** -24).all()) and bool((g == 0.5).all())
    before = [t.clone() for t in (flat, m, v)]
    for ps, gs in ((cut(flat, (0, 99, 200)), [g, g, g]), (cut(flat, (0, 0, 200)), [g, g, g]), (cut(flat), [g, flat[150:250], g]), (cut(flat), [g, m[:100], g])):
        with pytest.raises(ValueError, match='memory'):
            step(ps, gs)
    s = torch.zeros(2, 1, device=cuda_device).to(torch.float8_e8m0fnu)
    with pytest.raises(ValueError, match='memory'):
        adamw_step(cut(flat)[:2], [g, g], *([t.to(torch.float8_e4m3fn) for t in cut(x)[:2]] for x in (m, v)), [s, s], step=1)
    assert all(torch.equal(x, y) for x, y in zip(before, (flat, m, v)))
