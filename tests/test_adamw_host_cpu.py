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


# ---- states that the program replaces -------------------------------------------------------------------------------------
def _entry(name, make):
    def change(opt, p):
        opt.state[p][name] = make(opt.state[p][name])
    return change


def _emptied(opt, p):
    opt.state[p] = {}


def _cleared(opt, p):
    opt.state[p].clear()


def _deleted(opt, p):
    del opt.state[p]


def _other_memory(opt, p):
    opt.state[p]['exp_avg'].data = opt.state[p]['exp_avg'].data * 0.5


def _copied(opt, p):
    opt.state[p] = {k: v.clone() for k, v in opt.state[p].items()}
    opt.state[p]['exp_avg_sq'].mul_(9)


def _all_copied(opt, p):
    opt.state = type(opt.state)(dict, {k: {n: x.clone() for n, x in v.items()} for k, v in opt.state.items()})
    opt.state[p]['exp_avg'].mul_(-1)


CHANGES = {'exp_avg': _entry('exp_avg', torch.zeros_like), 'exp_avg_sq': _entry('exp_avg_sq', lambda x: x * 4), 'step': _entry('step', lambda x: torch.tensor(0.0)),
           'step further': _entry('step', lambda x: torch.tensor(1000.0)), 'same step': _entry('step', lambda x: x.clone()),
           'emptied': _emptied, 'cleared': _cleared, 'deleted': _deleted, 'other memory': _other_memory, 'copied': _copied, 'all copied': _all_copied}


@pytest.mark.parametrize('capturable', [False, True])
@pytest.mark.parametrize('change', sorted(CHANGES))
def test_replaced_states_are_taken(entries, change, capturable):
    x = Pair([5, 300, 7, 256], groups=2)
    if capturable:
        from pde_surrogate_amd import optim
        x.ours = optim.FusedAdamW(x.ours.param_groups, capturable=True)
    for _ in range(2):
        x.step()
    for k in (1, 2, 1):
        for ps, opt in x.both():
            CHANGES[change](opt, ps[k])
        x.step()
        x.step()
    x.step(which=(0, 3))
    x.step()
    for ps, opt in x.both():                       # while the parameter has no gradient
        CHANGES[change](opt, ps[3])
    x.step(which=(0, 1))
    x.step()
    a, b = x.ours.state_dict()['state'], x.torch.state_dict()['state']
    assert all(torch.allclose(a[k][n], b[k][n], rtol=1e-4, atol=1e-5) for k in b for n in b[k])


def test_a_count_that_is_a_number(entries):
    x = Pair([5, 300, 7], groups=1)
    x.step()
    for k in (0, 1, 2):
        x.ours.state[x.ps[k]]['step'] = 7
        x.torch.state[x.qs[k]]['step'] = torch.tensor(7.0)
    x.step()
    x.ours.state[x.ps[1]]['step'] = torch.tensor(3, dtype=torch.int64)
    x.torch.state[x.qs[1]]['step'] = torch.tensor(3.0)
    x.step()
    assert entries.launches == [3] * 3


def test_a_shared_count_that_changes_in_place_or_moves(entries):
    """parameters that are stepped together share one count here; in torch's optimiser each has its own"""
    x = Pair([5, 300, 7], groups=1)
    x.step()
    for move in (False, True):
        for ps, opt in x.both():
            for p in ps:
                if move:
                    opt.state[p]['step'].data = torch.tensor(40.0)
                else:
                    opt.state[p]['step'].fill_(11)
                if opt is x.ours:
                    break
        x.step()
    assert entries.launches == [3] * 3


@pytest.mark.parametrize('capturable', [False, True])
def test_states_that_are_taken_out_and_put_back(entries, capturable):
    """the tensors that a program holds are its own: nothing writes to them once others have taken their place"""
    x = Pair([5, 300, 7])
    if capturable:
        from pde_surrogate_amd import optim
        x.ours = optim.FusedAdamW(x.ours.param_groups, capturable=True)
    x.step()
    x.step()
    held = [opt.state[ps[1]] for ps, opt in x.both()]
    moment = [opt.state[ps[2]]['exp_avg'] for ps, opt in x.both()]
    copies = {k: v.clone() for k, v in held[0].items()}, moment[0].clone()
    for ps, opt in x.both():
        opt.state[ps[1]] = {}
        opt.state[ps[2]]['exp_avg'] = torch.ones(7)
    x.step()
    x.step()
    assert all(torch.equal(held[0][k], v) for k, v in copies[0].items() if k != 'step') and torch.equal(moment[0], copies[1])
    assert float(held[0]['step']) == 2
    for (ps, opt), h, m in zip(x.both(), held, moment):
        opt.state[ps[1]] = h
        opt.state[ps[2]]['exp_avg'] = m
    x.step()
    x.step()


def test_replaced_states_that_do_not_fit_are_refused_and_lose_nothing(entries):
    from pde_surrogate_amd import optim
    ps = params(5, 300, 7)
    opt = optim.FusedAdamW(ps)
    grads(ps, 1)
    opt.step()
    good = copy.deepcopy(opt.state_dict())
    weights = [p.detach().clone() for p in ps]
    first, second = opt.state[ps[0]], opt.state[ps[1]]['exp_avg']
    for change, match in ((lambda: opt.state[ps[1]].__setitem__('exp_avg', torch.zeros(7)), 'shape'),
                          (lambda: opt.state[ps[1]].pop('exp_avg_sq'), 'exp_avg_sq'), (lambda: opt.state[ps[1]].pop('step'), "'step'")):
        opt.state[ps[0]] = {k: v.clone() for k, v in first.items()}          # replaced as well, and fine
        kept = dict(opt.state[ps[1]])
        change()
        for _ in range(2):
            with pytest.raises(ValueError, match=match):
                opt.step()
        opt.state[ps[1]] = kept
        opt.state[ps[1]]['exp_avg'] = second
    assert all(torch.equal(p, w) for p, w in zip(ps, weights))
    now = opt.state_dict()
    assert all(torch.equal(now['state'][k][n], good['state'][k][n]) for k in range(3) for n in good['state'][k])
    other = optim.FusedAdamW(copy.deepcopy(ps))
    other.load_state_dict(good)
    for o in (opt, other):
        grads(o.param_groups[0]['params'], 2)
        o.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, other.param_groups[0]['params']))


def test_host_functions_on_states():
    """note and held: dictionaries that are changed and changed back, entries of the program's own, tensors that get other memory"""
    from pde_surrogate_amd.adamw import _host, _words
    host = _host()
    ps = params(3, 4)
    buf = torch.zeros(20)
    state = {p: {'step': torch.tensor(1.0), 'a': buf[5 * k:5 * k + 5]} for k, p in enumerate(ps)}
    known = [x for p in ps for x in (p, state[p], 'step', state[p]['step'], 'a', state[p]['a'], None)]
    dicts, tensors = [state[p] for p in ps], [state[p][k] for p in ps for k in ('step', 'a')]
    note, at = _words(1 + 2 + 8)
    host.note(state, dicts, tensors, at)

    def held():
        return host.held(state, known, dicts, tensors, at)
    assert held() and held()
    state[ps[1]]['mine'] = 3                       # entries of the program's own, in a state and beside them
    state['other'] = {}
    assert held() and held()
    keep = state[ps[0]]['a']
    state[ps[0]]['a'] = keep.clone()
    assert not held() and not held()
    state[ps[0]]['a'] = keep
    assert held()
    keep.data = keep.data.clone()
    assert not held()
    keep.data = buf[0:5]
    assert held()
    keep.data = buf[1:6]
    assert not held()
    keep.data = buf[0:5]
    for change, back in ((lambda: state.__setitem__(ps[0], dict(dicts[0])), lambda: state.__setitem__(ps[0], dicts[0])),
                         (lambda: state.__setitem__(ps[0], None), lambda: state.__setitem__(ps[0], dicts[0])),
                         (lambda: state[ps[1]].pop('step'), None), ):
        change()
        assert not held()
        if back:
            back()
            assert held()
    state[ps[1]] = {'step': known[10], 'a': known[12]}
    del state[ps[0]]
    assert not held()
    for bad in (lambda: host.held(state, known, dicts, tensors), lambda: host.held([], known, dicts, tensors, at), lambda: host.held(state, (), dicts, tensors, at),
                lambda: host.note(state, [3], [], at), lambda: host.note(state, [], [3], at), lambda: host.note(state, [], ())):
        with pytest.raises(TypeError):
            bad()


# ---- parameters that come to share memory ---------------------------------------------------------------------------------
def test_parameters_that_share_memory_after_a_step_are_refused(entries):
    from pde_surrogate_amd import optim
    ps = params(*[30 + k for k in range(12)])
    opt = optim.FusedAdamW([{'params': [p], 'lr': 1e-3 * (k + 1)} for k, p in enumerate(ps)])        # two launches
    grads(ps, 1)
    opt.step()
    assert entries.launches == [8, 4]
    whole = torch.randn(200)
    for a, b, mine, other in ((0, 1, slice(0, 30), slice(29, 60)), (0, 11, slice(50, 80), slice(40, 81)), (5, 7, slice(0, 35), slice(0, 37)),
                              (9, 2, slice(0, 39), slice(38, 70))):
        keep = ps[a].data, ps[b].data
        ps[a].data, ps[b].data = whole[mine], whole[other]
        before, states = whole.clone(), [x.clone() for x in opt.flat_state()['exp_avg']]
        for _ in range(2):
            with pytest.raises(RuntimeError, match='share their memory'):
                opt.step()
        assert torch.equal(whole, before) and all(torch.equal(x, y) for x, y in zip(states, opt.flat_state()['exp_avg']))
        assert float(opt.state[ps[a]]['step']) == 1 and len(entries.launches) == 2
        ps[a].data, ps[b].data = keep
    for k, p in enumerate(ps):                     # one behind the other without a gap, in any order
        at = (7 * k % 12) * 50
        p.data = torch.zeros(600)[at:at + 30 + k]
    opt.step()
    flat = torch.zeros(sum(p.numel() for p in ps))
    at = flat.numel()
    for p in ps:
        p.data = flat[at - p.numel():at]
        at -= p.numel()
    opt.step()
    assert float(opt.state[ps[3]]['step']) == 3


def test_stretches_of_memory():
    from pde_surrogate_amd.adamw import _host, _words

    def overlap(*lists):
        made = []
        for item, stretches in lists:
            (at, x), (n, y) = _words(len(stretches)), _words(len(stretches))
            for k, (start, size) in enumerate(stretches):
                at[k], n[k] = start, size
            made.append((x, y, len(stretches), item, at, n))
        return _host().overlap([m[:4] for m in made])
    assert not overlap() and not overlap((4, [])) and not overlap((4, [(8, 1), (12, 3), (24, 1)]))
    assert overlap((4, [(8, 1), (12, 3), (20, 1)])) and overlap((4, [(8, 4), (8, 4)])) and overlap((4, [(40, 1), (8, 9)]))
    assert not overlap((4, [(40, 1), (8, 8), (0, 0), (20, 0), (41, 0)])) and not overlap((2, [(40, 1), (8, 16)])) and overlap((2, [(40, 1), (8, 17)]))
    assert overlap((4, [(0, 1), (100, 1)]), (2, [(50, 2), (102, 1)])) and not overlap((4, [(0, 1), (100, 1)]), (2, [(50, 2), (104, 1)]))
    assert overlap((4, [((1 << 47) + 4, 1 << 39), (1 << 47, 2)])) and not overlap((4, [((1 << 47) + 4, 1 << 39), (1 << 47, 1)]))
    for bad in (lambda: _host().overlap(()), lambda: _host().overlap([3]), lambda: _host().overlap([(1, 2)]), lambda: _host().overlap()):
        with pytest.raises(TypeError):
            bad()


# ---- saving and loading ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('ours', [False, True])
def test_the_direction_is_part_of_a_saved_state(entries, ours):
    from pde_surrogate_amd import optim
    ps, qs, rs = params(5, 30), params(5, 30), params(5, 30)
    a, b = optim.FusedAdamW(ps, maximize=ours), optim.FusedAdamW(qs, maximize=not ours)
    grads(ps, 1)
    grads(qs, 1)
    a.step()
    b.step()
    keep = {k: v.clone() for k, v in b.state[qs[0]].items()}
    with pytest.raises(ValueError, match='maximize'):
        b.load_state_dict(a.state_dict())
    assert all(torch.equal(b.state[qs[0]][k], v) for k, v in keep.items())
    other = torch.optim.AdamW(rs, maximize=not ours)
    other.load_state_dict(copy.deepcopy(a.state_dict()))
    assert [g['maximize'] for g in other.param_groups] == [ours]
    for p, r in zip(ps, rs):
        r.data.copy_(p.data)
    for x, o in ((ps, a), (rs, other)):
        grads(x, 2)
        o.step()
    assert all(float((p - r).detach().abs().max()) <= 40 * 2.0 ** -24 * (1e-2 + float(p.detach().abs().max())) for p, r in zip(ps, rs))
    assert a.state_dict()['param_groups'][0]['maximize'] is ours
    # dictionaries without the entry, as they were saved before it was written, are taken as the optimiser's own
    sd = a.state_dict()
    del sd['param_groups'][0]['maximize']
    a.load_state_dict(sd)


def test_groups_with_choices_of_their_own_that_do_not_exist_are_refused(entries):
    from pde_surrogate_amd import optim
    ps = params(5, 6)
    for extra in (dict(maximize=True), dict(amsgrad=True)):
        with pytest.raises(ValueError, match=next(iter(extra))):
            optim.FusedAdamW([{'params': ps[:1]}, {'params': ps[1:], **extra}])
        opt = optim.FusedAdamW(ps[:1])
        with pytest.raises(ValueError, match=next(iter(extra))):
            opt.add_param_group({'params': ps[1:], **extra})
        assert len(opt.param_groups) == 1
    optim.FusedAdamW([{'params': ps, 'maximize': True, 'amsgrad': False}], maximize=True)


def test_hooks_on_saving_and_loading(entries):
    """as torch.optim documents them: a loading pre-hook sees the whole dictionary and may replace it, a post-hook sees the states that
    were loaded, hooks on saving see what is returned"""
    from pde_surrogate_amd import optim
    ps, qs = params(5, 30), params(5, 30)
    a, b = optim.FusedAdamW(ps), optim.FusedAdamW(qs)
    grads(ps, 1)
    a.step()
    seen = []
    a.register_state_dict_pre_hook(lambda o: seen.append('pre save'))

    def saved(o, sd):
        assert sd['state'][0]['step'] is not sd['state'][1]['step'] and sd['param_groups'][0]['maximize'] is False
        sd['mine'] = 'something'
        seen.append('post save')
    a.register_state_dict_post_hook(saved)

    def replaced(o, sd):
        assert o is b and set(sd['state']) == {0, 1} and sd['state'][0]['exp_avg'].shape == (5,) and sd['mine'] == 'something'
        seen.append('pre load')
        return {**sd, 'state': {0: {**sd['state'][0], 'exp_avg': sd['state'][0]['exp_avg'] * 2}, 1: sd['state'][1]}}
    b.register_load_state_dict_pre_hook(replaced)

    def loaded(o):
        assert torch.equal(o.state[qs[0]]['exp_avg'], a.state[ps[0]]['exp_avg'] * 2) and torch.equal(o.state[qs[1]]['exp_avg'], a.state[ps[1]]['exp_avg'])
        assert len(o.flat_state()['exp_avg']) == 1
        seen.append('post load')
    b.register_load_state_dict_post_hook(loaded)
    sd = a.state_dict()
    assert set(sd) == {'state', 'param_groups', 'mine'}
    for _ in range(2):
        b.load_state_dict(sd)
    assert seen == ['pre save', 'post save'] + ['pre load', 'post load'] * 2
    assert torch.equal(sd['state'][0]['exp_avg'], a.state[ps[0]]['exp_avg'])

    # a dictionary that cannot be taken, or a hook that fails: the optimiser is as it was, and the next one is taken as before
    grads(qs, 2)
    b.step()
    keep = [(k, {n: x.clone() for n, x in v.items()}) for k, v in b.state.items()]
    bad = copy.deepcopy(sd)
    bad['state'][1]['exp_avg'] = torch.zeros(3)
    with pytest.raises(ValueError, match='shape'):
        b.load_state_dict(bad)
    with pytest.raises(KeyError):
        b.load_state_dict({k: v for k, v in sd.items() if k != 'mine'})
    assert all(torch.equal(b.state[p][n], x) for p, st in keep for n, x in st.items())
    seen.clear()
    b.load_state_dict(sd)
    assert seen == ['pre load', 'post load'] and float(b.state[qs[0]]['step']) == 1


def test_a_dictionary_of_an_optimiser_whose_counts_are_numbers(entries):
    x = Pair([5, 30])
    x.step()
    x.ours.state[x.ps[0]]['step'] = 7
    assert x.ours.state_dict()['state'][0]['step'] == 7 and float(x.ours.state_dict()['state'][1]['step']) == 1


def test_an_optimiser_of_nothing_is_saved_and_loaded(entries):
    from pde_surrogate_amd import optim
    a, b = optim.FusedAdamW([{'params': [], 'lr': 0.5}]), optim.FusedAdamW([{'params': []}])
    b.load_state_dict(a.state_dict())
    b.step()
    assert b.param_groups[0]['lr'] == 0.5


# ---- memory ---------------------------------------------------------------------------------------------------------------
def _buffers(opt):
    return [len(v) for v in opt.flat_state().values()]


def test_buffers_of_states_that_have_moved_are_dropped(entries):
    from pde_surrogate_amd import optim
    import gc
    import weakref
    ps = [torch.nn.Parameter(torch.randn(8, 6, 3, 3)), torch.nn.Parameter(torch.randn(77))]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    a, b = optim.FusedAdamW(ps), optim.FusedAdamW(qs)
    gone = []
    for t in range(8):
        grads(qs, t)
        ps[0].grad = None
        ps[0].data = ps[0].data.to(memory_format=torch.channels_last if t % 2 else torch.contiguous_format)
        for p, q in zip(ps, qs):
            p.grad = q.grad.clone()
        a.step()
        b.step()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs))
        # the first buffers, in which the second parameter's states still are, and one more of each
        assert _buffers(a) == [1 if t == 0 else 2] * 2
        gone.append([weakref.ref(x[-1]) for x in a.flat_state().values()])
    gc.collect()
    assert [x[0]() is None and x[1]() is None for x in gone] == [False] + [True] * 6 + [False]
    # a state that is taken out again and again, and all of them at once
    for t in range(6):
        a.state[ps[1]] = {}
        a.step()
        assert _buffers(a) == [2] * 2
    a.state.clear()
    a.step()
    assert _buffers(a) == [1] * 2 and float(a.state[ps[0]]['step']) == 1


def test_a_changing_set_of_gradients_keeps_nothing(entries):
    """with counts on the device as well: only what a captured step works on is kept beside the states"""
    from pde_surrogate_amd import optim
    import gc
    import weakref
    ps = params(5, 30, 7)
    opt = optim.FusedAdamW(ps, capturable=True)
    counts = []
    for t in range(12):
        grads(ps, t, which=(0, 1, 2) if t % 2 else (0, t // 2 % 3))
        opt.step()
        counts += [weakref.ref(opt.state[p]['step']) for p in ps if p in opt.state]
    gc.collect()
    alive = {id(x()) for x in counts if x() is not None}
    assert alive == {id(opt.state[p]['step']) for p in ps}
    assert [float(opt.state[p]['step']) for p in ps] == [12, 8, 8]

    # a captured step's counts and buffers stay (the stand-in computes at once what a graph would compute when it is replayed)
    grads(ps, 0)
    opt.step()
    entries.capturing = True
    opt.step()
    entries.capturing = False
    kept = [weakref.ref(x) for x in [opt.state[p]['step'] for p in ps] + [x for v in opt.flat_state().values() for x in v]]
    opt.load_state_dict(opt.state_dict())
    opt.state.clear()
    grads(ps, 1, which=(1,))
    opt.step()
    gc.collect()
    assert all(x() is not None for x in kept)
    late = [weakref.ref(x) for x in [opt.state[ps[1]]['step']] + [x for v in opt.flat_state().values() for x in v]]
    opt.load_state_dict(opt.state_dict())
    gc.collect()
    assert all(x() is None for x in late) and all(x() is not None for x in kept)


# ---- the C entries --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('at', [159, 160, 161, 400])
def test_a_bad_entry_anywhere_in_a_list_is_refused_before_anything_is_launched(at):
    """every call is rejected on the host (a launch takes 160 tensors, and the ones in front are fine)"""
    import ctypes
    from pde_surrogate_amd import _lib
    L = _lib.lib()
    for address, size, want in ((0, 10, -1), (4098, 10, -3), (4096, -1, -1), (4096, 1 << 40, -1)):
        grads_, sizes = (ctypes.c_ulonglong * 401)(*[4096] * 401), (ctypes.c_longlong * 401)(*[10] * 401)
        grads_[at], sizes[at] = address, size
        assert L.pdes_grad_norm(grads_, sizes, 401, 0, 2, 4096, 0, None) == want
        assert L.pdes_clip_grads(grads_, sizes, 401, 0, 2, 4096, 1.0, 4096, None) == want
        # without a limit nothing is read, and the list is checked all the same
        assert L.pdes_clip_grads(grads_, sizes, 401, 0, 2, 4096, float('inf'), 4096, None) == want
    sizes = (ctypes.c_longlong * 401)(*[1 << 32] * 401)                  # 2^40 and more together
    assert L.pdes_grad_norm((ctypes.c_ulonglong * 401)(*[4096] * 401), sizes, 401, 0, 2, 4096, 0, None) == -1


def test_everything_at_once(entries):
    """a gradient less, one more, another memory order, a moved parameter and a replaced moment before one step"""
    x = Pair([5, 300, 7, 256, 64], groups=2)
    for ps, opt in x.both():
        ps[4].data = ps[4].data.view(8, 8)
    x.step(which=(0, 1, 4))
    for t in range(3):
        for ps, opt in x.both():
            ps[4].grad = None
            ps[4].data = ps[4].data.t().contiguous().t() if t % 2 == 0 else ps[4].data.contiguous()
            opt.param_groups[t % 2]['params'].append(opt.param_groups[1 - t % 2]['params'].pop(0))
            opt.state[ps[1]]['exp_avg'] = opt.state[ps[1]]['exp_avg'] + 1
        x.step(which=(1, 2 + t % 2, 4))
        x.step()


@pytest.mark.parametrize('capturable', [False, True])
def test_a_count_that_is_a_number_while_its_parameter_has_no_gradient(entries, capturable):
    from pde_surrogate_amd import optim
    ps = params(5, 30, 7)
    opt = optim.FusedAdamW(ps, capturable=capturable)
    grads(ps, 1)
    opt.step()
    opt.state[ps[2]]['step'] = 20
    for t in range(2):
        grads(ps, 2 + t, which=(0, 1))
        opt.step()
    assert opt.state[ps[2]]['step'] == 20
    grads(ps, 4)
    opt.step()
    assert [float(opt.state[p]['step']) for p in ps] == [4, 4, 21]


def test_copies_are_saved_and_loaded(entries):
    """a copied and a pickled optimiser step, save and load as the one they come from"""
    import pickle
    from pde_surrogate_amd import optim
    ps = params(5, 30)
    a = optim.FusedAdamW(ps)
    grads(ps, 1)
    a.step()
    for x, b in (copy.deepcopy((ps, a)), pickle.loads(pickle.dumps((ps, a)))):
        sd = b.state_dict()
        assert all(torch.equal(sd['state'][k]['exp_avg'], a.state[p]['exp_avg']) for k, p in enumerate(ps))
        b.load_state_dict(a.state_dict())
        keep = [p.detach().clone() for p in ps]
        c = optim.FusedAdamW(ps)
        c.load_state_dict(a.state_dict())
        for opt, y in ((b, x), (c, ps)):
            grads(y, 2)
            opt.step()
        assert all(torch.equal(p, q) for p, q in zip(ps, x))
        for p, k in zip(ps, keep):
            p.data.copy_(k)
