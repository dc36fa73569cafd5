"""AdamW over many tensors in one launch (``ml_adamw_step``), moments in 32 bits or in the 8-bit blocks of ``monoloco_amd.fp8``.

For the loop a caller owns (``outputs = model(inputs)``; ``loss.backward()``; ``optimizer.step()``): the reference builds torch's Adam
there (monoloco/train/trainer.py:128-131).  ``HipTrainer`` has its own Adam inside the library and does not need this one."""
from array import array
from operator import attrgetter

import torch

from .. import _lib
from .._lib import MonolocoHipError
from ..fp8 import BLOCK, CODES, DTYPES, SCALES, _need, _run

_T = torch.Tensor
_dtype = attrgetter('dtype')


def _address(a):
    return a.buffer_info()[0]


def state_scales(numel, device):
    """Scales of the 8-bit moments of a tensor of `numel` elements: row 0 for exp_avg, row 1 for the root of exp_avg_sq; all 1."""
    return torch.ones((2, -(-numel // BLOCK)), device=device).to(SCALES)


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, scales=None, *, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, seed=0):
    """One AdamW step in place: ``step`` counts from 1, all tensors of one type (fp32, bf16, fp16) and device, contiguous,
    none twice and none sharing memory with another (refused).

    Without ``scales`` the moments are fp32 tensors like the parameters.  With ``scales`` (one (2, ceil(numel / 128)) tensor of e8m0 for
    each parameter, see ``state_scales``) they are e4m3 codes: exp_avgs of the first moment, exp_avg_sqs of the ROOT of the second, both
    rounded stochastically from ``seed``, the step, the tensor's place in the lists and the element (the same call gives the same bits).
    Refused while its stream is captured: the step's number is part of the launch."""
    k = len(params)
    _need(len(grads) == k and len(exp_avgs) == k and len(exp_avg_sqs) == k and (scales is None or len(scales) == k),
          "adamw_step: %d parameters, %d gradients, %d and %d moments", k, len(grads), len(exp_avgs), len(exp_avg_sqs))
    _need(int(step) >= 1, "adamw_step: steps are counted from 1, got %r", step)
    if not k:
        return
    dt, index = params[0].dtype, params[0].get_device()
    if not params[0].is_cuda:
        raise MonolocoHipError("adamw_step runs on HIP devices only, got a tensor on %s (there is no CPU fallback)" % (params[0].device,))
    _need(dt in DTYPES, "adamw_step: parameters are fp32, bf16 or fp16, got %s", dt)
    mdt = torch.float32 if scales is None else CODES
    # (whole lists at a time: for a network of 38 tensors a check per tensor and property costs more than the launch)
    sizes = list(map(_T.numel, params))
    for what, ts, want in (('parameters', params, dt), ('gradients', grads, dt), ('first moments', exp_avgs, mdt), ('second moments', exp_avg_sqs, mdt)):
        if set(map(_dtype, ts)) != {want}:
            raise ValueError("adamw_step: %s parameters take %s gradients and %s moments, got %s as %s" % (dt, dt, mdt, sorted(map(str, set(map(_dtype, ts)))), what))
        if set(map(_T.get_device, ts)) != {index}:
            raise ValueError("adamw_step: the %s are not all on cuda:%d" % (what, index))
        if ts is not params and list(map(_T.numel, ts)) != sizes:
            raise ValueError("adamw_step: the %s are not of their parameters' sizes" % what)
        if not all(map(_T.is_contiguous, ts)):
            if ts is not grads:
                raise ValueError("adamw_step: the %s have to be contiguous" % what)
            grads = [g.contiguous() for g in grads]
    if scales is not None:
        for s, n in zip(scales, sizes):
            if not (s.dtype == SCALES and s.get_device() == index and s.is_contiguous() and tuple(s.shape) == (2, -(-n // BLOCK))):
                raise ValueError("adamw_step: the scales of %d elements are a contiguous (2, %d) of %s on cuda:%d, got %s %s on %s"
                                 % (n, -(-n // BLOCK), SCALES, index, tuple(s.shape), s.dtype, s.device))
    ps, gs, ms, vs = (array('Q', map(_T.data_ptr, ts)) for ts in (params, grads, exp_avgs, exp_avg_sqs))
    ss = array('Q', map(_T.data_ptr, scales)) if scales is not None else None
    numel = array('q', sizes)
    _run(index, _lib.load().ml_adamw_step, k, _address(numel), _address(ps), _address(gs),
         DTYPES[dt], _address(ms), _address(vs), None if ss is None else _address(ss), int(step), float(lr), float(betas[0]), float(betas[1]), float(eps),
         float(weight_decay), int(seed) & 0xffffffff)
    torch.autograd.graph.increment_version(params)   # (LocoModel re-packs its engine when a parameter's version moved)


def _check_group(g):
    """A parameter group, given or loaded, that asks for this step and no other one."""
    missing = [k for k in ('lr', 'betas', 'eps', 'weight_decay') if k not in g]
    _need(not missing, "AdamW: a group without %s", ', '.join(missing))
    _need(g.get('state_bits', 32) in (8, 32), "AdamW: moments have 8 or 32 bits, not %r", g.get('state_bits'))
    _need(g['lr'] >= 0 and g['eps'] >= 0 and g['weight_decay'] >= 0 and all(0 <= b < 1 for b in g['betas']),
          "AdamW: lr, eps and weight_decay are not negative, betas are in [0, 1)")
    for flag in ('maximize', 'amsgrad'):
        _need(not g.get(flag), "AdamW: %s is not supported", flag)
    _need(g.get('decoupled_weight_decay', True) or not g['weight_decay'], "AdamW: the weight decay is decoupled from the gradient, a group asks for the other kind")


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW``'s arguments, groups, schedulers and state_dict on ``adamw_step``; groups that ask for ``maximize``, ``amsgrad``
    or a decay through the gradient are refused.

    ``state_bits=8`` keeps the moments as e4m3 blocks (2 + 1/64 bytes per parameter instead of 8); ``seed`` is their rounding's: each
    tensor of an optimizer has random bits of its own, two optimizers take two seeds.
    Parameters that got no gradient are left as they are, each counts its own steps."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32, seed=0):
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits, seed=int(seed)))

    def add_param_group(self, param_group):
        _check_group({**self.defaults, **param_group})
        super().add_param_group(param_group)

    def _state(self, p, bits):
        s = self.state[p]
        if not s:
            s['step'] = 0
            for key in ('exp_avg', 'exp_avg_sq'):
                s[key] = torch.zeros(p.shape, dtype=torch.float32, device=p.device).to(torch.float32 if bits == 32 else CODES)
            if bits == 8:
                s['scales'] = state_scales(p.numel(), p.device)
        return s

    @staticmethod
    def _in_place(lists, places):
        """The lists with tensors without elements wherever a place has none (the library skips them, but counts them)."""
        out = []
        for ts in lists:
            none = ts[0].new_empty(ts[0].shape[:1] + (0,) if ts is lists[4] else 0)
            full = [none] * (places[-1] + 1)
            for i, t in zip(places, ts):
                full[i] = t
            out.append(full)
        return out

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for place, group in enumerate(self.param_groups):
            bits, kinds = group['state_bits'], {}
            for p in group['params']:
                kinds.setdefault((p.device, p.dtype), []).append(p)
            for kind, ps in enumerate(kinds.values()):
                # random bits go by seed, step and place in the call: a seed of its own for every call of a step, and (below) a place for
                # every tensor that does not depend on which of the others have a gradient
                seed = (group['seed'] + 0x9e3779b9 * place + 0x85ebca6b * kind) & 0xffffffff
                calls = {}
                for i, p in enumerate(ps):
                    if p.grad is None:
                        continue
                    _need(not p.grad.is_sparse, "AdamW: sparse gradients are not supported")
                    s = self._state(p, bits)
                    calls.setdefault(s['step'] + 1, []).append((i, p, s))
                for step, found in calls.items():
                    lists = [[p for _, p, _ in found], [p.grad for _, p, _ in found], [s['exp_avg'] for _, _, s in found], [s['exp_avg_sq'] for _, _, s in found]]
                    if bits == 8:
                        lists.append([s['scales'] for _, _, s in found])
                        if found[-1][0] >= len(found):
                            lists = self._in_place(lists, [i for i, _, _ in found])
                    adamw_step(*lists[:4], lists[4] if bits == 8 else None, step=step, lr=float(group['lr']), betas=group['betas'], eps=group['eps'],
                               weight_decay=group['weight_decay'], seed=seed)
                    for _, _, s in found:
                        s['step'] = step
        return loss

    def load_state_dict(self, state_dict):
        """As torch's, but the moments keep the types they were saved in (the base class casts them to the parameters').  A state_dict of
        ``torch.optim.AdamW`` loads, too (moments in 32 bits); what asks for another rule is refused before anything changes."""
        own = [{k: g[k] for k in ('state_bits', 'seed')} for g in self.param_groups]
        saved_groups = state_dict['param_groups']
        for mine, saved in zip(own, saved_groups):
            bits = saved.get('state_bits', 32)
            _need(bits == mine['state_bits'], "AdamW: the saved moments have %d bits, this optimizer's %d", bits, mine['state_bits'])
        for g in saved_groups:
            _check_group(g)
            need = {'step', 'exp_avg', 'exp_avg_sq'} | ({'scales'} if g.get('state_bits', 32) == 8 else set())
            for i in g['params']:
                keys = set(state_dict['state'].get(i) or need)
                _need(need <= keys and 'mu_product' not in keys, "AdamW: the state of another optimizer: %s", sorted(keys))
        super().load_state_dict(state_dict)
        ids = [i for g in saved_groups for i in g['params']]
        for g, mine in zip(self.param_groups, own):
            for k, v in mine.items():
                g.setdefault(k, v)
        for i, p in zip(ids, [p for g in self.param_groups for p in g['params']]):
            saved = state_dict['state'].get(i)
            if saved:
                state = self.state[p]      # (what a caller keeps there beside stays as the base class loaded it)
                state['step'] = int(saved['step'])
                for k in ('exp_avg', 'exp_avg_sq', 'scales'):
                    if k in saved:
                        v = saved[k].detach().to(p.device).clone()
                        state[k] = v.float() if v.dtype in DTYPES else v
