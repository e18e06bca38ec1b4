"""optim.Muon beside the framework: schedules, groups and checkpoints."""

import copy

import pytest
import torch

from parallax_amd import lr_schedule, optim

GPU = pytest.mark.gpu
DEVICES = ['cpu', pytest.param('cuda', marks=GPU)]


def _leaves(dev, seed=0):
    g = torch.Generator().manual_seed(seed)

    def leaf(*s):
        return torch.nn.Parameter(torch.randn(*s, generator=g).to(dev))

    return dict(mat=leaf(20, 30), vec=leaf(30), head=leaf(10, 30),
                table=leaf(50, 8))


def _grads(ps, seed):
    g = torch.Generator().manual_seed(seed)
    for name, p in ps.items():
        if name == 'table':
            ids = torch.tensor([3, 7])
            p.grad = torch.sparse_coo_tensor(
                ids[None], torch.randn(2, 8, generator=g),
                (50, 8)).to(p.device)
        else:
            p.grad = torch.randn(p.shape, generator=g).to(p.device)


def _groups(ps, **kw):
    return [dict(params=[ps['mat'], ps['vec'], ps['table']], **kw),
            dict(params=[ps['head']], muon=False, adam_lr=1e-2)]


@pytest.mark.parametrize('dev', DEVICES)
def test_a_schedule_reaches_every_parameter(dev):
    """Steps from zero moments: Adam's and Muon's are proportional to their
    rates, up to a rounding of the parameter (2^-24 of up to 5)."""
    moved = {}
    for part in (1.0, 0.5, 0.0):
        ps = _leaves(dev)
        opt = optim.Muon(_groups(ps))
        lr_schedule.set_lr(opt, 0.02 * part)
        _grads(ps, 1)
        before = {k: p.detach().clone() for k, p in ps.items()}
        opt.step()
        moved[part] = {k: p.detach() - before[k] for k, p in ps.items()}
    for k, whole in moved[1.0].items():
        assert whole.abs().max() > 1e-5, k
        assert torch.allclose(moved[0.5][k] * 2, whole, rtol=1e-5,
                              atol=4 * 5 * 2.0 ** -24), k
        assert not moved[0.0][k].any(), k


def test_rates_of_groups():
    ps = _leaves('cpu')
    opt = optim.Muon(_groups(ps, lr=0.1), lr=0.02)
    extra = torch.nn.Parameter(torch.zeros(3))
    opt.add_param_group(dict(params=[extra], lr=0.4))
    rate = opt._adam_lr
    assert [rate(g) for g in opt.param_groups] == [3e-4, 1e-2, 3e-4]
    sched = torch.optim.lr_scheduler.LambdaLR(opt, lambda i: 1 / (1 + i))
    opt.step()
    sched.step()
    assert [rate(g) for g in opt.param_groups] == [1.5e-4, 5e-3, 1.5e-4]
    zero = optim.Muon([torch.nn.Parameter(torch.zeros(3))], lr=0.0)
    assert rate(zero.param_groups[0]) == 3e-4


def test_a_schedule_goes_on_from_a_checkpoint():
    def run(ps, opt, steps):
        for i in steps:
            lr_schedule.set_lr(opt, 0.02 / (1 + i))
            _grads(ps, i)
            opt.step()

    a = _leaves('cpu')
    oa = optim.Muon(_groups(a))
    run(a, oa, range(2))
    state = copy.deepcopy(oa.state_dict())
    lacks = dict(state, param_groups=[
        {k: v for k, v in g.items() if k != 'base_lr'}
        for g in state['param_groups']])
    others = []
    for s in (state, lacks):
        b = {k: torch.nn.Parameter(p.detach().clone()) for k, p in a.items()}
        ob = optim.Muon(_groups(b))
        ob.load_state_dict(copy.deepcopy(s))
        run(b, ob, range(2, 4))
        others.append(b)
    run(a, oa, range(2, 4))
    for b in others:
        for k in a:
            assert torch.equal(a[k], b[k]), k
