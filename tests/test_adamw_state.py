"""AdamW's groups and state on the CPU: what it cannot honour is refused, with nothing changed (no GPU: no step is launched)."""
import copy

import pytest
import torch

from monoloco_amd.train import AdamW


def params(k=2):
    return [torch.nn.Parameter(torch.full((3,), float(i))) for i in range(k)]


def stepped(cls, **kw):
    ps = params()
    o = cls(ps, lr=0.5, **kw)
    for p in ps:
        p.grad = torch.ones(3)
    o.step()
    return o.state_dict()


def refused(own, saved, text):
    before = copy.deepcopy(own.state_dict())
    with pytest.raises(ValueError, match=text):
        own.load_state_dict(copy.deepcopy(saved))
    assert own.state_dict() == before and not own.state


@pytest.mark.parametrize('cls,kw,text', [(torch.optim.AdamW, dict(maximize=True), 'maximize'), (torch.optim.AdamW, dict(amsgrad=True), 'amsgrad'),
                                         (torch.optim.Adam, dict(maximize=True), 'maximize'), (torch.optim.Adam, dict(weight_decay=0.1), 'decay'),
                                         (torch.optim.SGD, dict(momentum=0.9), 'betas'), (torch.optim.NAdam, {}, 'another'), (torch.optim.Adamax, {}, 'another')])
def test_states_of_other_rules_are_refused(cls, kw, text):
    refused(AdamW(params(), lr=0.25), stepped(cls, **kw), text)


def test_the_last_group_counts_too():
    ps = params()
    o = torch.optim.AdamW([{'params': ps[:1]}, {'params': ps[1:], 'maximize': True}])
    qs = params()
    refused(AdamW([{'params': qs[:1]}, {'params': qs[1:]}]), o.state_dict(), 'maximize')


def test_states_of_the_same_rule_load():
    for cls, kw in ((torch.optim.AdamW, {}), (torch.optim.Adam, {}), (torch.optim.AdamW, dict(foreach=True, weight_decay=0.1))):
        saved = stepped(cls, **kw)
        o = AdamW(params(), state_bits=32, seed=5)
        o.load_state_dict(saved)
        g = o.param_groups[0]
        assert g['lr'] == 0.5 and g['weight_decay'] == saved['param_groups'][0]['weight_decay'] and (g['state_bits'], g['seed']) == (32, 5)
        for i, p in enumerate(g['params']):
            assert o.state[p]['step'] == 1 and all(torch.equal(o.state[p][k], saved['state'][i][k]) for k in ('exp_avg', 'exp_avg_sq'))


def test_what_a_caller_keeps_beside_the_moments_loads():
    a = AdamW(params())
    for p in a.param_groups[0]['params']:
        a._state(p, 32)['average'] = p.detach().clone() + 1
    b = AdamW(params())
    b.load_state_dict(copy.deepcopy(a.state_dict()))
    for p, q in zip(a.param_groups[0]['params'], b.param_groups[0]['params']):
        assert set(b.state[q]) == {'step', 'exp_avg', 'exp_avg_sq', 'average'} and torch.equal(b.state[q]['average'], a.state[p]['average'])


@pytest.mark.parametrize('kw,text', [(dict(maximize=True), 'maximize'), (dict(amsgrad=True), 'amsgrad'), (dict(decoupled_weight_decay=False), 'decay'),
                                     (dict(state_bits=16), 'bits'), (dict(betas=(0.9, 1.0)), 'betas'), (dict(lr=-1.0), 'lr')])
def test_groups_are_checked(kw, text):
    with pytest.raises(ValueError, match=text):
        AdamW([{'params': params(1)}, {'params': params(1), **kw}])
    o = AdamW(params(1))
    with pytest.raises(ValueError, match=text):
        o.add_param_group({'params': params(1), **kw})
    assert len(o.param_groups) == 1
    o.add_param_group({'params': params(1), 'state_bits': 8, 'maximize': False, 'name': 'last'})
    assert o.param_groups[1]['name'] == 'last' and o.param_groups[1]['seed'] == 0


def test_no_two_tensors_share_random_bits(monkeypatch):
    """The bits follow from (seed, step, place in the call): over groups, types and parameters that lag behind (no gradient for some steps) no
    two tensors ever meet with the same three, and a tensor's place does not depend on which of the others have gradients."""
    import monoloco_amd.train.adamw as A
    calls = []

    def record(ps, gs, ms, vs, scales, *, step, seed, **_):
        assert len(ps) == len(gs) == len(ms) == len(vs) == len(scales)
        calls.extend((seed, step, i, p) for i, p in enumerate(ps) if p.numel())

    monkeypatch.setattr(A, 'adamw_step', record)
    ps = params(6) + [torch.nn.Parameter(torch.zeros(3, dtype=torch.bfloat16)) for _ in range(3)]
    groups = [[ps[0], ps[1], ps[6], ps[2]], [ps[3], ps[7]], [ps[4], ps[8], ps[5]]]
    o = AdamW([{'params': g} for g in groups], state_bits=8, seed=77)
    seen, places = {}, {}
    for it in range(6):
        for k, p in enumerate(ps):
            p.grad = None if (k + it) % 3 == 0 else torch.ones_like(p)
        calls.clear()
        o.step()
        assert {id(c[3]) for c in calls} == {id(p) for p in ps if p.grad is not None} and len(calls) == 6
        for seed, step, i, p in calls:
            assert seen.setdefault((seed, step, i), id(p)) == id(p)
            assert places.setdefault(id(p), (seed, i)) == (seed, i)
            assert o.state[p]['step'] == step
    assert places[id(ps[0])] == (77, 0) and places[id(ps[1])] == (77, 1)       # the first tensors: as adamw_step with the same seed
    assert all(0 <= s < 1 << 32 for s, _ in places.values())


def test_shared_memory_is_refused(hip_lib):
    """Decided on the host, before any HIP call (no pointer here is ever used: every call is refused)."""
    import ctypes

    def call(text, eight=False, dtype=0, **move):
        n = 3
        numel = [128, 0, 300]
        at = {k: [0x10000 * (1 + 4 * j), 0, 0x10000 * (2 + 4 * j)] for j, k in enumerate(('p', 'g', 'm', 'v', 's'))}
        for k, (i, a) in move.items():
            at[k][i] = a
        arr = lambda k: (ctypes.c_void_p * n)(*[a or None for a in at[k]])  # noqa: E731
        assert hip_lib.ml_adamw_step(n, (ctypes.c_int64 * n)(*numel), arr('p'), arr('g'), dtype, arr('m'), arr('v'), arr('s') if eight else None, 1, 1e-3, 0.9,
                                     0.999, 1e-8, 0.01, 0, None) == 1
        assert text in hip_lib.ml_ops_last_error().decode(), hip_lib.ml_ops_last_error()

    p0, p2, m0, s0 = 0x10000, 0x20000, 0x90000, 0x110000
    both = 'given twice, or tensors share memory (0 and 2)'
    for eight in (False, True):
        call(both, eight, p=(2, p0))                              # the same parameter
        call(both, eight, p=(2, p0 + 128 * 4 - 4))                # its last element
        call(both, eight, p=(2, p0 - 300 * 4 + 4))                # its first one
        call(both, eight, dtype=1, p=(2, p0 + 128 * 2 - 2))
        call(both, eight, v=(2, p0 + 8))
        call('tensors share memory (0 and 0)', eight, m=(0, p0))
        call('gradient 0 shares memory with what the step writes of tensor 2', eight, g=(0, p2))
        call('gradient 2 shares memory with what the step writes of tensor 2', eight, g=(2, p2 + 4))
        call('gradient 2 shares memory with what the step writes of tensor 0', eight, g=(2, m0 - 300 * 4 + 1))
    call(both, True, s=(2, s0))                                   # the same scales
    call(both, True, s=(2, s0 + 1))
    call(both, True, s=(2, m0 + 127))


def test_library_refusals_are_value_errors(hip_lib):
    """Wrong arguments raise ValueError, whoever finds them."""
    from monoloco_amd import _lib
    assert hip_lib.ml_sum_rows(None, -1, 1, None, 0, None) == 1
    with pytest.raises(ValueError, match='bad type') as e:
        _lib.check_ops(1)
    assert isinstance(e.value, _lib.MonolocoHipError)
    with pytest.raises(_lib.MonolocoHipError) as e:
        _lib.check_ops(2)
    assert not isinstance(e.value, ValueError)
