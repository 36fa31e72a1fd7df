"""GPU tests of what FusedAdamW does with groups, states and memory that a program changes between steps, with the kernels (the decisions
themselves: tests/test_adamw_host_cpu.py)."""
import math

import numpy as np
import pytest
import torch

import adamw_util as au

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def dev():
    assert torch.cuda.is_available()
    return torch.device('cuda:0')


def _params(dev, sizes, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter((torch.randn(n, generator=g) * 0.05).to(dtype).to(dev)) for n in sizes]


def _grads(params, seed, which=None):
    g = torch.Generator().manual_seed(seed)
    for k, p in enumerate(params):
        x = (torch.randn(p.shape, generator=g) * 10.0 ** (-(k % 4))).to(p.dtype).to(p.device)
        p.grad = x if which is None or k in which else None


@pytest.mark.parametrize('bits,dtype,master', [(32, torch.float32, False), (32, torch.bfloat16, True), (8, torch.float32, False), (8, torch.bfloat16, True)])
def test_groups_and_states_that_a_program_changes(dev, bits, dtype, master):
    """the same changes to an optimiser that has stepped all along and to one that is made anew and loads the changed dictionary: bit for
    bit the same steps"""
    from pde_surrogate_amd import optim
    sizes = [5, 300, 1024, 4097]
    kw = dict(state_bits=bits, master_weights=master, clip_norm=1.0, seed=5)
    ps = _params(dev, sizes, dtype)
    a = optim.FusedAdamW([{'params': ps[:2], 'lr': 1e-3}, {'params': ps[2:], 'lr': 3e-2, 'weight_decay': 0.3}], **kw)
    for t in range(2):
        _grads(ps, t)
        a.step()

    def moved():                                            # the list keeps its order: so do the random sequences of the 8-bit states
        a.param_groups[1]['params'].insert(0, a.param_groups[0]['params'].pop())

    def replaced():
        a.param_groups[0] = dict(a.param_groups[0], lr=5e-2)

    def moment():
        st = a.state[ps[3]]
        name = 'exp_avg' if bits == 32 else 'exp_avg_scale'
        st[name] = st[name] * 2

    def count():
        a.state[ps[1]]['step'] = torch.tensor(50.0)

    def memory():
        for st in a.state.values():                         # states that were away from the device
            for v in st.values():
                v.data = v.data.cpu()

    def emptied():
        a.state[ps[0]] = {}

    for t, change in enumerate((moved, replaced, moment, count, memory, emptied)):
        change()
        qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
        by = dict(zip(ps, qs))
        b = optim.FusedAdamW([dict(g, params=[by[p] for p in g['params']]) for g in a.param_groups], **kw)
        b.load_state_dict(a.state_dict())
        for s in range(2):
            _grads(ps, 10 * t + s)
            for p, q in zip(ps, qs):
                q.grad = p.grad.clone()
            a.step()
            b.step()
            for p, q in zip(ps, qs):
                assert torch.equal(p, q), change.__name__
                assert float(a.state[p]['step']) == float(b.state[q]['step'])
                for k in a.state[p]:
                    assert a.state[p][k].device == b.state[q][k].device
                    assert torch.equal(a.state[p][k].reshape(-1).view(torch.uint8), b.state[q][k].reshape(-1).view(torch.uint8)), (change.__name__, k)


def test_a_captured_step_whose_states_are_replaced_meanwhile(dev):
    """the graph goes on with the states it was captured with, in memory that nothing else gets"""
    from pde_surrogate_amd import optim
    ps, qs = _params(dev, [700, 5000]), _params(dev, [700, 5000])
    a, b = (optim.FusedAdamW(x, lr=1e-2, capturable=True) for x in (ps, qs))
    for x, opt in ((ps, a), (qs, b)):
        _grads(x, 0)
        opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    a.load_state_dict(a.state_dict())
    a.state.clear()
    a.zero_grad(set_to_none=False)
    for p in ps:
        p.grad.zero_()
    keep = [p.detach().clone() for p in ps]
    a.step()
    for p, k in zip(ps, keep):
        p.data.copy_(k)
    filler = [torch.full((4096,), 3.0, device=dev) for _ in range(50)]
    for t in range(1, 4):
        _grads(qs, t)
        for p, q in zip(ps, qs):
            p.grad.copy_(q.grad)
        graph.replay()
        b.step()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    assert all((x == 3.0).all() for x in filler) and float(a.state[ps[0]]['step']) == 1


def test_counts_and_buffers_outlive_another_streams_work(dev, monkeypatch):
    """every eager step tells the allocator which stream works on them"""
    from pde_surrogate_amd import optim
    told, real = [], torch.Tensor.record_stream
    monkeypatch.setattr(torch.Tensor, 'record_stream', lambda self, s: (told.append((self.data_ptr(), s.cuda_stream)), real(self, s))[1])
    ps = _params(dev, [700, 50])
    opt = optim.FusedAdamW(ps, capturable=True)
    _grads(ps, 0)
    opt.step()
    torch.cuda.synchronize()
    told.clear()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        opt.step()
    torch.cuda.synchronize()
    assert {x for x, y in told if y == s.cuda_stream} == {opt.state[ps[0]]['step'].data_ptr()} | {v[0].data_ptr() for v in opt.flat_state().values()}


def test_parameters_that_come_to_share_memory(dev):
    from pde_surrogate_amd import optim
    ps = _params(dev, [1000, 1000, 300])
    opt = optim.FusedAdamW(ps)
    _grads(ps, 0)
    opt.step()
    keep = ps[1].data
    ps[1].data = ps[0].data
    before = [p.detach().clone() for p in ps]
    with pytest.raises(RuntimeError, match='share their memory'):
        opt.step()
    assert all(torch.equal(p, x) for p, x in zip(ps, before)) and float(opt.state[ps[0]]['step']) == 1
    ps[1].data = keep
    opt.step()
    assert float(opt.state[ps[0]]['step']) == 2


@pytest.mark.parametrize('capturable', [False, True])
def test_a_capture_that_is_refused_changes_nothing(dev, capturable):
    from pde_surrogate_amd import optim
    ps = [torch.nn.Parameter(torch.randn(8, 6, 3, 3, device=dev)), torch.nn.Parameter(torch.randn(77, device=dev))]
    opt = optim.FusedAdamW(ps, capturable=capturable)
    _grads(ps, 0)
    opt.step()
    ps[0].grad = None
    ps[0].data = ps[0].data.to(memory_format=torch.channels_last)
    _grads(ps, 1)
    before = [p.detach().clone() for p in ps]
    states = [x.clone() for v in opt.flat_state().values() for x in v]
    with pytest.raises(RuntimeError, match='eagerly' if capturable else 'capturable'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    assert all(torch.equal(p, x) for p, x in zip(ps, before))
    assert all(torch.equal(x, y) for x, y in zip(states, [x for v in opt.flat_state().values() for x in v]))
    want = [torch.nn.Parameter(x) for x in before]
    other = optim.FusedAdamW(want)
    other.load_state_dict(opt.state_dict())
    for p, q in zip(ps, want):
        q.grad = p.grad.clone()
    opt.step()
    other.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, want))
