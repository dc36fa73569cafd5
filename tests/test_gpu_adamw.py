"""monoloco_amd.train.AdamW / adamw_step against the formula in 64 bits.

Tolerances, derived before the first run (u = 2^-24): constants are rounded once (u), every operation adds u.  m and v: 4 u of the sum of
their terms' magnitudes.  The update lr / bc1 * m / den: 16 u of size * (|b1 m| + |(1 - b1) g|) / den; p: 3 u |p| more, and half a step of its
type.  8-bit codes: m' is off by 4 u, that is less than 2^-16 of a step, so that a code differs from the 64-bit one where the 16 random
bits meet the fraction that closely: fewer than one in 1000, by one step."""
import copy

import pytest
import torch

import ref8 as R
from monoloco_amd.network.architectures import LocoModel
from monoloco_amd.train import AdamW, adamw_step, state_scales

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HYPER = dict(lr=2e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.05)
SHAPES = [(1,), (3, 5), (128,), (129,), (0,), (64, 64), (4095,), (4097,), (7, 1000), (2048,), (16,)]


def make(seed, shapes, dtype):
    g = torch.Generator().manual_seed(seed)
    p = [(0.1 * torch.randn(s, generator=g)).to(dtype) for s in shapes]
    gr = [(1e-2 * torch.randn(s, generator=g) * torch.exp(torch.randn(s, generator=g))).to(dtype) for s in shapes]
    m = [3e-3 * torch.randn(s, generator=g) for s in shapes]
    r = [(1e-2 * torch.randn(s, generator=g)).abs() + 1e-4 for s in shapes]
    return p, gr, m, r


def dev(ts, d):
    return [t.to(d) for t in ts]


def check_p(got, p, g, m, v, step, dtype, hyper=HYPER):
    want, m2, v2, am, size = R.adamw(p.double(), g.double(), m, v, step, **hyper)
    tol = 16 * U * size * am + 3 * U * p.double().abs() + half(dtype) * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert bool(((got.cpu().double() - want).abs() <= tol).all())
    return m2, v2, am


def half(t):
    return torch.finfo(t).eps / 2


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('step', [1, 7, 100000])
def test_step_32(cuda_device, dtype, step):
    shapes = SHAPES * 7            # 77 tensors: more than one launch holds
    p, g, m, r = make(step, shapes, dtype)
    v = [t * t for t in r]
    P, G, M, V = (dev(t, cuda_device) for t in (p, g, m, v))
    adamw_step(P, G, M, V, step=step, **HYPER)
    for i in range(len(p)):
        m2, v2, am = check_p(P[i], p[i], g[i], m[i].double(), v[i].double(), step, dtype)
        assert bool(((M[i].cpu().double() - m2).abs() <= 4 * U * am).all()) and bool(((V[i].cpu().double() - v2).abs() <= 5 * U * v2).all())
        assert torch.equal(G[i].cpu(), g[i])


def encode(ts, root=False):
    q, s = [], []
    for t in ts:
        n = t.numel()
        if n == 0:
            q.append(t.to(F8)), s.append(torch.zeros((0,), dtype=torch.uint8))
            continue
        c, b = R.quantize(torch.nn.functional.pad(t.reshape(-1), (0, -n % 128)).view(-1, 128))
        q.append(c.reshape(-1)[:n].view(t.shape).float().to(F8)), s.append(b.reshape(-1).to(torch.uint8))
    return q, s


def decode(q, b):
    n = q.numel()
    return (q.float().double().reshape(-1) * R.scale_values(b).repeat_interleave(128)[:n]).view(q.shape)


@pytest.mark.parametrize('dtype', TYPES)
def test_step_8(cuda_device, dtype):
    shapes, step, seed = SHAPES * 6, 9, 0x12345678
    p, g, m, r = make(3, shapes, dtype)
    (qm, sm), (qr, sr) = encode(m), encode(r)
    P, G, M, V = (dev(t, cuda_device) for t in (p, g, qm, qr))
    S = [torch.stack([a, b]).view(E8).to(cuda_device) for a, b in zip(sm, sr)]
    adamw_step(P, G, M, V, S, step=step, seed=seed, **HYPER)
    differ = total = 0
    for i in range(len(p)):
        n = p[i].numel()
        m0, r0 = decode(qm[i], sm[i]), decode(qr[i], sr[i])
        m2, v2, am = check_p(P[i], p[i], g[i], m0, r0 * r0, step, dtype)
        u = R.bits(seed, step, i, n) if n else torch.zeros(0, dtype=torch.int64)
        for row, (code, x, bits) in enumerate(((M[i], m2, u & 0xffff), (V[i], v2.sqrt(), u >> 16))):
            if not n:
                continue
            want, wb = R.stochastic(x.reshape(-1), bits, row == 1)
            got, gb = code.cpu().float().double().reshape(-1), S[i].view(torch.uint8).cpu()[row].long()
            assert torch.equal(gb, wb)
            off = (got - want).abs()
            # (m2 is off by 4 u am, which a cancelling sum makes more than 4 u of itself)
            assert bool((off <= R.step_of(torch.maximum(want.abs(), got.abs())) * 1.001).all())
            differ, total = differ + int((off > 0).sum()), total + n
    assert differ <= 1e-3 * total, (differ, total)


def test_rounding_is_unbiased_and_seeded(cuda_device):
    """b1 = b2 = 0.999 and a gradient that repeats: rounding to nearest would never move a moment.  Stochastic rounding keeps the mean of m
    exactly on its course.  A rounding's variance is at most step * move, relative 2^-3 * 0.001, and decays with 0.999^2: in all at most
    2^-3 * 0.001 * 500 = 0.0625, a deviation of 0.25 per element, 0.0028 for the mean of 8192, 0.014 for five of them."""
    n = 128 * 64
    g = torch.full((n,), 0.01, device=cuda_device)
    p, m, v, s = torch.zeros(n, device=cuda_device), torch.zeros(n, device=cuda_device).to(F8), torch.zeros(n, device=cuda_device).to(F8), state_scales(n, cuda_device)
    for step in range(1, 4001):
        adamw_step([p], [g], [m], [v], [s], step=step, lr=0.0, betas=(0.999, 0.999), weight_decay=0.0, seed=5)
    want = 1 - 0.999 ** 4000
    mean = float((m.float() * s[0].float().repeat_interleave(128)).mean()) / 0.01
    root = float((v.float() * s[1].float().repeat_interleave(128)).mean()) / 0.01
    assert abs(mean - want) < 0.014
    assert abs(root - want ** 0.5) < 0.05     # E[r^2] = v + var: at rest 0.001 (E[v] - g^2) = step * move <= 2^-3 * 0.0005 * |g^2 - r^2| / r,
                                              # relative 2^-4 of a deviation of at most 0.5: v is pushed up by 0.03, its root by 0.015
    a = [t.clone() for t in (m, v, s)]
    ms = []
    for seed in (1, 1, 2):
        x = [t.clone() for t in a]
        adamw_step([p], [g], [x[0]], [x[1]], [x[2]], step=5, lr=0.0, betas=(0.999, 0.999), seed=seed)
        ms.append(x[0].view(torch.uint8).clone())
    assert torch.equal(ms[0], ms[1]) and not torch.equal(ms[0], ms[2])


def test_small_second_moments_stay(cuda_device):
    """A positive second moment far below its block's largest never becomes 0, and a block of zeros stays zeros."""
    n = 256
    g = torch.zeros(n)
    g[0], g[1:128] = 1.0, 1e-9
    p, m, v, s = torch.zeros(n, device=cuda_device), torch.zeros(n, device=cuda_device).to(F8), torch.zeros(n, device=cuda_device).to(F8), state_scales(n, cuda_device)
    adamw_step([p], [g.to(cuda_device)], [m], [v], [s], step=1, seed=3)
    c = v.view(torch.uint8).cpu()
    assert bool((c[1:128] == 1).all()) and not c[128:].any() and s.view(torch.uint8)[:, 1].tolist() == [127, 127]
    assert torch.isfinite(p).all() and not p[128:].any()


def test_not_finite(cuda_device):
    n = 300
    for bits in (32, 8):
        for bad in (float('nan'), float('inf')):
            g = torch.full((n,), 0.01)
            g[200] = bad
            p = torch.ones(n, device=cuda_device)
            m, v, s = torch.zeros(n, device=cuda_device), torch.zeros(n, device=cuda_device), None
            if bits == 8:
                m, v, s = m.to(F8), v.to(F8), [state_scales(n, cuda_device)]
            adamw_step([p], [g.to(cuda_device)], [m], [v], s, step=1)
            ok = torch.ones(n, dtype=torch.bool)
            ok[200] = False
            assert torch.equal(torch.isfinite(p).cpu(), ok)            # this step: its own element
            blk = torch.zeros(n, dtype=torch.bool)
            blk[128:256] = bits == 8
            blk[200] = True
            assert torch.equal(torch.isfinite(m.float()).cpu(), ~blk)  # 8 bits: the block's scale is NaN


def test_views_and_untouched_surroundings(cuda_device):
    """Tensors cut out of one buffer at odd offsets: what lies between them stays."""
    sizes, gap = [5, 130, 1, 4096, 77], 3
    total = sum(n + gap for n in sizes) + 1
    g0 = torch.Generator().manual_seed(1)
    for bits in (32, 8):
        flat = torch.randn(total, generator=g0)
        P = flat.to(cuda_device)
        M, V = (torch.full((total,), 0.5, device=cuda_device).to(torch.float32 if bits == 32 else F8) for _ in range(2))
        at, views = 1, []
        for n in sizes:
            views.append(slice(at, at + n))
            at += n + gap
        G = [0.01 * torch.randn(n, generator=g0) for n in sizes]
        scales = [state_scales(n, cuda_device) for n in sizes] if bits == 8 else None
        adamw_step([P[s] for s in views], dev(G, cuda_device), [M[s] for s in views], [V[s] for s in views], scales, step=2, **HYPER)
        for s, g in zip(views, G):
            check_p(P[s], flat[s], g, torch.full(g.shape, 0.5).double(), torch.full(g.shape, 0.5 if bits == 32 else 0.25).double(), 2, torch.float32)
        keep = torch.ones(total, dtype=torch.bool)
        for s in views:
            keep[s] = False
        assert torch.equal(P.cpu()[keep], flat[keep]) and bool((M.float().cpu()[keep] == 0.5).all()) and bool((V.float().cpu()[keep] == 0.5).all())


def test_refusals(cuda_device):
    def t(n=4, d=torch.float32):
        return torch.zeros(n, device=cuda_device, dtype=d)
    p = t()
    for args, kw in ((([p], [t(4, torch.bfloat16)], [t()], [t()]), {}), (([p], [t()], [t(4, torch.bfloat16)], [t()]), {}), (([p], [t(5)], [t()], [t()]), {}),
                     (([p, p], [t(), t()], [t(), t()], [t(), t()]), {}), (([p], [t()], [p], [t()]), {}), (([p], [torch.zeros(4)], [t()], [t()]), {}),
                     (([t(8)[::2]], [t()], [t()], [t()]), {}), (([p], [t()], [t()], [t()]), dict(scales=[state_scales(4, cuda_device)])),
                     (([p], [t()], [t().to(F8)], [t().to(F8)]), dict(scales=[state_scales(400, cuda_device)])), (([t(4, torch.float64)],) * 4, {})):
        with pytest.raises(ValueError):
            adamw_step(*args, step=1, **kw)
    graph, side = torch.cuda.CUDAGraph(), t()
    args = ([p], [t()], [t()], [t()])
    with torch.cuda.graph(graph):
        side.add_(1)
        with pytest.raises(Exception, match='captured'):
            adamw_step(*args, step=1)
    graph.replay()
    torch.cuda.synchronize()
    assert float(side[0]) == 1 and not p.any()


def test_optimizer_like_torch(cuda_device):
    """The class over groups, a schedule, parameters without gradients and mixed types: torch.optim.AdamW's trajectory in fp64."""
    shapes = [(40, 30), (40,), (9, 40), (9,), (300,)]
    g0 = torch.Generator().manual_seed(4)
    ps = [torch.nn.Parameter(torch.randn(s, generator=g0).to(cuda_device)) for s in shapes]
    qs = [torch.nn.Parameter(p.detach().cpu().double()) for p in ps]
    opts = []
    for cls, t in ((AdamW, ps), (torch.optim.AdamW, qs)):
        o = cls([{'params': t[:2], 'lr': 1e-2}, {'params': t[2:], 'weight_decay': 0.2}], lr=3e-3, betas=(0.8, 0.95))
        opts.append((o, torch.optim.lr_scheduler.StepLR(o, 3, 0.5)))
    for it in range(8):
        for i, (p, q) in enumerate(zip(ps, qs)):
            p.grad = q.grad = None
            if i != 4 or it % 2:
                g = torch.randn(p.shape, generator=g0)
                p.grad, q.grad = g.to(cuda_device), g.double()
        for o, sch in opts:
            o.step()
            sch.step()
        if it == 4:       # through a state_dict into a new optimizer
            fresh = AdamW([{'params': ps[:2], 'lr': 1e-2}, {'params': ps[2:], 'weight_decay': 0.2}], lr=3e-3, betas=(0.8, 0.95))
            fresh.load_state_dict(copy.deepcopy(opts[0][0].state_dict()))
            sch = torch.optim.lr_scheduler.StepLR(fresh, 3, 0.5)
            sch.load_state_dict(opts[0][1].state_dict())
            opts[0] = (fresh, sch)
    for p, q in zip(ps, qs):   # 8 steps of at most 1e-2 * 5: 8 * (12 + 3) u of values of order 1
        assert float((p.detach().cpu().double() - q.detach()).abs().max()) < 8 * 20 * U * 6


def test_optimizer_8_bits_state_dict(cuda_device):
    p = torch.nn.Parameter(torch.randn(1000, generator=torch.Generator().manual_seed(1)).bfloat16().to(cuda_device))
    o = AdamW([p], lr=1e-2, state_bits=8, seed=3)
    for _ in range(3):
        p.grad = torch.randn(1000, generator=torch.Generator().manual_seed(2)).bfloat16().to(cuda_device)
        o.step()
    p2 = torch.nn.Parameter(p.detach().clone())
    o2 = AdamW([p2], lr=1e-2, state_bits=8, seed=3)
    o2.load_state_dict(copy.deepcopy(o.state_dict()))
    for k in ('exp_avg', 'exp_avg_sq', 'scales'):
        assert o2.state[p2][k].dtype == o.state[p][k].dtype and torch.equal(o2.state[p2][k].view(torch.uint8), o.state[p][k].view(torch.uint8))
    p2.grad = p.grad.clone()
    o.step(), o2.step()
    assert torch.equal(p, p2)
    with pytest.raises(ValueError):
        AdamW([p2], state_bits=32).load_state_dict(o.state_dict())
    twin = copy.deepcopy(o)                     # a copy keeps what it needs for its next step
    q = twin.param_groups[0]['params'][0]
    q.grad = p.grad.clone()
    o.step(), twin.step()
    assert torch.equal(p, q)


def test_optimizer_takes_over_from_torch(cuda_device):
    g0 = torch.Generator().manual_seed(9)
    p = torch.nn.Parameter(torch.randn(300, generator=g0).to(cuda_device))
    q = torch.nn.Parameter(p.detach().clone())
    a, b = torch.optim.AdamW([p], lr=1e-2), AdamW([q], lr=1e-2)
    for it in range(4):
        g = torch.randn(300, generator=g0).to(cuda_device)
        if it == 2:
            q.data.copy_(p.data)
            b.load_state_dict(copy.deepcopy(a.state_dict()))
            assert b.state[q]['step'] == 2 and b.param_groups[0]['state_bits'] == 32
        for t, o in ((p, a), (q, b)):
            t.grad = g.clone()
            o.step()
    # two steps of the same formula in fp32 from the same state: (16 u * 1e-2 + 4 u |p|) each, on both sides
    assert float((p - q).abs().max()) <= 4 * (16 * U * 1e-2 * 4 + 4 * U * 5)


def test_module_sees_the_step(cuda_device):
    """LocoModel re-packs its engine and its train-mode twin after a step of this optimizer, as after torch's."""
    torch.manual_seed(0)
    model = LocoModel(34, 9, 256, p_dropout=0.0, num_stage=1).to(cuda_device)
    other = copy.deepcopy(model)
    x = torch.randn(64, 34, generator=torch.Generator().manual_seed(1)).to(cuda_device)
    outs = []
    for net, cls in ((model, AdamW), (other, torch.optim.AdamW)):
        opt = cls(net.parameters(), lr=1e-2, weight_decay=0.01)
        net.eval()
        before = net(x).clone()
        net.train()
        for _ in range(2):
            opt.zero_grad()
            net(x).square().mean().backward()
            opt.step()
        net.eval()
        after = net(x)
        assert not torch.equal(before, after)
        outs.append(after)
    # the first Adam steps are lr * sign(g) where |g| is far above eps: elements whose gradient is rounding noise may differ by 2 lr
    assert float((outs[0] - outs[1]).norm() / outs[1].norm()) < 0.05
