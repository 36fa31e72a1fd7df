"""What FusedAdamW decides on the host, on CPU tensors (tests/adamw_host.py): torch.optim.AdamW does the same to the same optimiser
and is compared with.  Both round an fp32 update of lr at most in another order: 40 roundings of 2^-24 of (10 lr + |w|) a step.  The first
moment is a sum of terms of up to max |g| together (under 6 here), which may cancel: each side rounds constants, products and sum, 4 of
2^-24 of that a step; the second moment's terms are positive, and 5 roundings a step of it are under 1e-5 for ten steps."""
import copy

import pytest
import torch

from adamw_host import grads, host_only, params


@pytest.fixture(scope='module', autouse=True)
def _built():
    from pde_surrogate_amd import build
    build.build(verbose=False)                 # (nothing to do where everything is built)


@pytest.fixture
def entries(monkeypatch):
    return host_only(monkeypatch)


class Pair:
    """the same groups, gradients and treatment for FusedAdamW and torch.optim.AdamW"""

    def __init__(self, sizes, groups=1, **kw):
        from pde_surrogate_amd import optim
        self.ps, self.qs = params(*sizes), params(*sizes)
        made = []
        for x in (self.ps, self.qs):
            cut = -(-len(x) // groups)
            made.append([{'params': x[k:k + cut], 'lr': 1e-3 * (1 + 10 * j), 'weight_decay': 0.3 * j}
                         for j, k in enumerate(range(0, len(x), cut))])
        self.ours, self.torch = optim.FusedAdamW(made[0], **kw), torch.optim.AdamW(made[1], foreach=False, **kw)
        self.t = 0

    def both(self):
        return (self.ps, self.ours), (self.qs, self.torch)

    def step(self, which=None):
        self.t += 1
        for x, opt in self.both():
            grads(x, self.t, which)
            opt.step()
        for k, (p, q) in enumerate(zip(self.ps, self.qs)):
            lr = max(g['lr'] for g in self.ours.param_groups)
            assert float((p - q).detach().abs().max()) <= self.t * 40 * 2.0 ** -24 * (10 * lr + float(q.detach().abs().max())), f'parameter {k}, step {self.t}'
            st, other = self.ours.state.get(p), self.torch.state.get(q)
            assert bool(st) == bool(other)
            if st:
                assert float(st['step']) == float(other['step']), f'parameter {k}, step {self.t}'
                for name, atol in (('exp_avg', self.t * 8 * 2.0 ** -24 * 6), ('exp_avg_sq', 1e-12)):
                    assert torch.allclose(st[name], other[name], rtol=1e-5, atol=atol), f'{name} of parameter {k}, step {self.t}'


def test_the_stand_in_is_adamw(entries):
    x = Pair([5, 300, 1, 256], groups=2)
    for _ in range(4):
        x.step()
    assert entries.launches == [4] * 4


# ---- groups that the program changes --------------------------------------------------------------------------------------
def test_a_parameter_that_moves_to_another_group(entries):
    x = Pair([5, 300, 7, 256], groups=2)
    x.step()
    for _, opt in x.both():
        opt.param_groups[1]['params'].insert(0, opt.param_groups[0]['params'].pop())
    x.step()
    for _, opt in x.both():
        opt.param_groups[0]['params'].append(opt.param_groups[1]['params'].pop(0))
    x.step()


def test_a_group_that_another_dictionary_replaces(entries):
    x = Pair([5, 300, 7, 256], groups=2)
    x.step()
    for _, opt in x.both():
        opt.param_groups[0] = dict(opt.param_groups[0], lr=7e-2, weight_decay=0.01)
    x.step()
    for _, opt in x.both():
        opt.param_groups[0]['lr'] = 1e-4
    x.step()
    for _, opt in x.both():
        opt.param_groups = [dict(g, lr=g['lr'] * 2) for g in opt.param_groups]
    x.step()
