"""AdamW over many tensors at once, and clipping by the gradients' common norm.

    opt = optim.FusedAdamW(model.parameters(), lr=1e-3, weight_decay=0.01)                 # 32-bit states
    opt = optim.FusedAdamW(model.parameters(), lr=1e-3, state_bits=8, clip_norm=1.0)       # 8-bit states, clipped
    norm = optim.clip_grad_norm_(model.parameters(), 1.0)                                  # for any optimiser

Any list of fp32, bf16 or fp16 parameters on one GPU takes part, whichever module they belong to: `optim.Adam` needs one HIP
network's flat buffer for its one-launch step, `FusedAdamW` takes the tensors as they are, up to 96 in a launch.  The
kernels are csrc/multi_tensor.hip; the arithmetic is fp32 with one rounding per operation (include/pdes_hip.h:
pdes_adamw_step, and the one exception), the norm's sum is fp64 in a fixed order, so equal inputs give equal bits.
"""
import ctypes
import math
from array import array
from collections import defaultdict

import torch

from . import _lib

BLOCK = 256                   # PDES_MT_BLOCK: every tensor's state starts at a multiple of it; elements that share a scale
_CLASSES = 8                  # PDES_MT_CLASSES
_ROWS = 256                   # PDES_MT_ROWS
_HYPER_BYTES = 288            # PDES_MT_HYPER_BYTES
_LARGEST = 2.0 ** 128 - 2.0 ** 104            # the largest fp32 number
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class MtTensor(ctypes.Structure):
    _fields_ = [('n', ctypes.c_longlong), ('block0', ctypes.c_longlong), ('cls', ctypes.c_int), ('ordinal', ctypes.c_int)]


class AdamWClass(ctypes.Structure):
    _fields_ = [(k, ctypes.c_double) for k in ('lr', 'beta1', 'beta2', 'eps', 'weight_decay')] + \
               [('step', ctypes.c_longlong), ('step_dev', ctypes.c_void_p), ('lr_dev', ctypes.c_void_p)]


class AdamWState(ctypes.Structure):
    _fields_ = [(k, ctypes.c_void_p) for k in ('exp_avg', 'exp_avg_sq', 'exp_avg_scale', 'rms_scale', 'low')] + \
               [('blocks', ctypes.c_longlong), ('norm_rows', ctypes.c_void_p), ('norm_out', ctypes.c_void_p),
                ('hyper', ctypes.c_void_p), ('limit', ctypes.c_float), ('dtype', ctypes.c_int), ('bits', ctypes.c_int),
                ('maximize', ctypes.c_int), ('seed', ctypes.c_uint)]


_host_module = None
# the current stream's handle: torch.cuda.current_stream makes an object of it first, 1.8 us of the 17 that a step of one tensor takes
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None)


def _stream(device):
    return _raw_stream(device.index) if _raw_stream is not None else _lib.stream_ptr(device)


def _host():
    """_tensor_list.so (csrc/tensor_list.cpp); there is no fallback"""
    global _host_module
    if _host_module is None:
        try:
            from . import _tensor_list
        except ImportError as e:
            raise RuntimeError(f'pde_surrogate_amd/_tensor_list.so cannot be loaded ({e}): build it with `python -m pde_surrogate_amd.build`') from e
        _host_module = _tensor_list
    return _host_module


def _dense(t):
    """whether the elements of `t` fill one stretch of memory, each once (any order of the dimensions)"""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != want:
            return False
        want *= size
    return True


def _same_order(a, b):
    """whether element k of a's memory is element k of b's"""
    return all(n == 1 or x == y for n, x, y in zip(a.shape, a.stride(), b.stride()))


def _order(t):
    """the dimensions of a dense tensor from the outermost in memory to the innermost; those of one element have no place"""
    return tuple(sorted((d for d in range(t.dim()) if t.shape[d] != 1), key=lambda d: -t.stride(d)))


def _check_tensor(t, what):
    if t.layout != torch.strided:
        raise RuntimeError(f'{what}: sparse tensors are not supported')
    if t.dtype not in _DTYPES:
        raise RuntimeError(f'{what}: expected float32, bfloat16 or float16, got {t.dtype}')
    if not t.is_cuda:
        raise RuntimeError(f'pde_surrogate_amd runs on an MI355X only: {what} is a CPU tensor (there is no CPU fallback; '
                           'move tensors to cuda)')


def _overlap(stretches):
    """whether two of the (address, bytes) stretches have bytes in common"""
    end = 0
    for start, size in sorted(x for x in stretches if x[1]):
        if start < end:
            return True
        end = start + size
    return False


def _words(n):
    """n zeroed 64-bit numbers for the C entries, and their address"""
    a = array('Q', bytes(8 * n))
    return a, a.buffer_info()[0]


def _limit(x):
    """a limit as fp32: only infinity is none"""
    return x if x == math.inf else min(x, _LARGEST)


def _norm_rows(lists, kind, device, stream):
    """pdes_grad_norm over [(element type, address of the addresses, address of the sizes, how many)]"""
    rows = torch.empty(_ROWS, dtype=torch.float64, device=device)
    for k, (dtype, ptrs, sizes, count) in enumerate(lists):
        rc = _lib.lib().pdes_grad_norm(ptrs, sizes, count, dtype, kind, rows.data_ptr(), int(k > 0), stream)
        _lib.check(rc, 'pdes_grad_norm')
    return rows


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_ for parameters on one GPU: returns the norm of all gradients taken as one vector (0-d
    fp32 on the device) and multiplies the gradients in place by min(1, max_norm / (norm + 1e-6)), without synchronising.
    norm_type is 2 (summed in fp64) or infinity.  max_norm = inf finds the norm only.  Where the factor is 1 the gradients
    are read once and not written.  A gradient that is not dense (an expanded one) or shares memory with another is refused.
    error_if_nonfinite waits for the norm and raises, with the gradients as they were, if it is not finite."""
    params = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    max_norm, norm_type = float(max_norm), float(norm_type)
    if norm_type not in (2.0, math.inf):
        raise ValueError(f'clip_grad_norm_: norm_type {norm_type} is not supported (2 or inf)')
    if not max_norm >= 0.0:
        raise ValueError(f'clip_grad_norm_: max_norm {max_norm} must not be negative')
    n = len(params)
    (ptrs, ptr_at), (sizes, size_at) = _words(3 * n), _words(3 * n)
    *counts, index, bad, shared = _host().gradients(params, ptr_at, size_at)
    if bad >= 0:
        g = params[bad].grad
        _check_tensor(g, 'a gradient')
        if not _dense(g):
            raise RuntimeError('clip_grad_norm_: a gradient is not dense')
        raise RuntimeError(f'clip_grad_norm_: gradients on cuda:{index} and {g.device}')
    if shared:
        raise ValueError('clip_grad_norm_: two gradients share their memory')
    lists = [(dtype, ptr_at + 8 * n * dtype, size_at + 8 * n * dtype, count) for dtype, count in enumerate(counts) if count]
    if not lists:
        return torch.tensor(0.0)
    device = torch.device('cuda', index)
    kind = 2 if norm_type == 2.0 else 0
    with _lib.device_guard(device):
        stream = _stream(device)
        rows = _norm_rows(lists, kind, device, stream)
        norm = torch.empty((), dtype=torch.float32, device=device)

        def clip(dtype, ptrs, sizes, count, limit):
            rc = _lib.lib().pdes_clip_grads(ptrs, sizes, count, dtype, kind, rows.data_ptr(), limit, norm.data_ptr(), stream)
            _lib.check(rc, 'pdes_clip_grads')

        if error_if_nonfinite or max_norm == math.inf:
            clip(*lists[0], math.inf)
            if error_if_nonfinite and not math.isfinite(float(norm)):
                raise RuntimeError(f'the norm of order {norm_type} of the gradients is not finite, so they cannot be clipped; with '
                                   'error_if_nonfinite=False they are multiplied by the factor that it gives')
        if max_norm != math.inf:
            for x in lists:
                clip(*x, _limit(max_norm))
            _host().changed(params, True)
    return norm


def _check_lr(lr, device):
    if lr.dim() or lr.dtype != torch.float32 or lr.device != device:
        raise ValueError(f'lr as a tensor has to be a 0-d float32 tensor on {device}, got {lr.dim()}-d {lr.dtype} on {lr.device}')


class _Arena:
    """state buffers of a list of parameters of one element type, each from a multiple of BLOCK elements on"""

    def __init__(self, dtype, blocks, bits, master, device):
        self.dtype, self.blocks = dtype, blocks

        def zeros(n, t):
            return torch.zeros(n, dtype=t, device=device)
        n = blocks * BLOCK
        if bits == 32:
            self.bufs = {'exp_avg': zeros(n, torch.float32), 'exp_avg_sq': zeros(n, torch.float32)}
        else:
            self.bufs = {'exp_avg_q': zeros(n, torch.uint8).view(torch.float8_e4m3fn), 'exp_avg_scale': zeros(blocks, torch.float32),
                         'rms_q': zeros(n, torch.uint8).view(torch.float8_e4m3fn), 'rms_scale': zeros(blocks, torch.float32)}
        if master and dtype == torch.bfloat16:
            self.bufs['low'] = zeros(n, torch.int16)
        self.names = {'step', *self.bufs}
        self.stream = _stream(device)

    def views(self, p, block0):
        """{name: the part of it that belongs to p}: in p's shape and order where there is one value per element"""
        n, blocks = p.numel(), -(-p.numel() // BLOCK)
        out = {}
        for name, buf in self.bufs.items():
            if name.endswith('_scale'):
                out[name] = buf[block0:block0 + blocks]
            elif name.endswith('_q'):
                out[name] = buf[block0 * BLOCK:(block0 + blocks) * BLOCK]
            else:
                out[name] = buf.as_strided(p.shape, p.stride(), block0 * BLOCK) if n else buf[:0].view(p.shape)
        return out


class _Launch:
    """one pdes_adamw_step call: parameters of one arena in up to eight classes"""

    def __init__(self, arena, members, classes):
        # members: (parameter, its class, block0, ordinal, its state's order); classes: (param_group, step tensor)
        self.arena, self.count = arena, len(members)
        # on the host, counts are incremented through numpy: a tenth of the time of a tensor's addition
        self.classes = [(g, step, None if step.is_cuda else step.numpy()) for g, step in classes]
        self.params, self.like = [m[0] for m in members], [m[4] for m in members]
        self.table = (AdamWClass * len(classes))()
        self.state = st = AdamWState()
        self.tensors = array('q')                          # pdes_mt_tensor: n, block0, cls | ordinal << 32
        for p, cls, block0, ordinal, _ in members:
            self.tensors.extend((p.numel(), block0, cls | ordinal << 32))
        # filled anew by every step; the sizes are what the parameters are held to
        (self.ptrs, self.ptr_at), (self.grads, self.grad_at) = _words(self.count), _words(self.count)
        self.sizes = self.tensors[::3]
        self.size_at, self.tensor_at, self.total = self.sizes.buffer_info()[0], self.tensors.buffer_info()[0], sum(self.sizes)
        for name, key in (('exp_avg', 'exp_avg'), ('exp_avg_sq', 'exp_avg_sq'), ('exp_avg', 'exp_avg_q'), ('exp_avg_sq', 'rms_q'),
                          ('exp_avg_scale', 'exp_avg_scale'), ('rms_scale', 'rms_scale'), ('low', 'low')):
            if key in arena.bufs:
                setattr(st, name, arena.bufs[key].data_ptr())
        st.blocks, st.dtype = arena.blocks, _DTYPES[arena.dtype]


class _Reordered(Exception):
    """a parameter's memory has another order than its state's"""


class _Ungraded(Exception):
    """a parameter of the plan has no gradient any more"""


class _Plan:
    """the launches of a step, for as long as the same parameters of the same groups have gradients and no state is replaced"""

    def __init__(self, launches, groups):
        self.launches = launches
        self.stretches = [(x.ptr_at, x.size_at, x.count, x.params[0].element_size()) for x in launches]
        self.groups = [x for g in groups for x in (g, len(g['params']))]       # (the launches' constants come from these dictionaries)
        self.params = [p for g in groups for p in g['params']]
        self.mask = bytes(p.grad is not None for p in self.params)


class FusedAdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay, torch.optim.AdamW's update) over any fp32 / bf16 / fp16 parameters of one GPU.

    state_bits      32: exp_avg and exp_avg_sq in fp32, in the parameter's shape: a torch.optim.AdamW state_dict loads here and
                    the other way round.  8: both moments in 8 bits (e4m3, the second one as its square root) with an fp32
                    scale for each 256 elements and stochastic rounding: 2.06 bytes per element instead of 8.
    master_weights  bf16 parameters keep the 16 bits that bf16 cuts off (state 'low', 2 bytes per element), so that the step
                    works on fp32 weights; a parameter that the program overwrites is taken as it is, to half of its last
                    place.  Without it a bf16 / fp16 parameter is rounded to nearest after every step, as torch does.
    clip_norm       gradients are multiplied by min(1, clip_norm / (norm + 1e-6)) as the step reads them, the norm taken over
                    all gradients of the step; `.grad` stays as it is, `grad_norm` is the norm (0-d tensor on the device).
    capturable      step counts live on the device, so that a step may be captured into a graph; take one eager step first, which
                    makes the states.  `lr` may be a 0-d fp32 device tensor then, read at every replay (a number is captured).
    seed            of the stochastic rounding: equal seeds, parameters and gradients give equal bits.

    `state` may be changed as torch.optim.AdamW's may: entries replaced, a state emptied or put back.  Parameters of a group that have
    taken equally many steps share one 'step' tensor, which an in-place change alters for all of them.

    A gradient of another memory order than its parameter's is copied into the parameter's first; every parameter has to be
    dense, and no two may share memory.  Parameters without a gradient are left out of a step, as in torch.  `amsgrad`, sparse
    and complex parameters are not offered.  A gradient that is not finite spoils the elements it belongs to and no others,
    unless a finite clip_norm lets it into the common factor: an infinite norm makes that 0 (all other gradients count as zeros in
    that step), a NaN makes it NaN, and with it every parameter, as torch's clipping and step do.
    With 8-bit states eps under 2^-100 counts as 2^-100, and blocks whose largest value is under that are held as zeros; they
    belong to stretches of the parameter's memory, so a parameter keeps the order of its dimensions there for good.

    A graph captured from a step holds the states it was captured with: capture again after load_state_dict, and after a step
    in which other parameters had gradients or states were replaced.  The states and counts that such a graph writes to are kept for as
    long as the optimiser."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, master_weights=False,
                 clip_norm=None, maximize=False, capturable=False, seed=0):
        if state_bits not in (8, 32):
            raise ValueError(f'state_bits {state_bits} is not supported (8 or 32)')
        if clip_norm is not None and not float(clip_norm) >= 0.0:
            raise ValueError(f'clip_norm {clip_norm} must not be negative')
        if not 0 <= int(seed) < 1 << 32:
            raise ValueError(f'seed {seed} is not in [0, 2^32)')
        self.state_bits, self.master_weights, self.maximize = state_bits, bool(master_weights), bool(maximize)
        self.clip_norm, self.capturable, self.seed = None if clip_norm is None else float(clip_norm), bool(capturable), int(seed)
        self.grad_norm = None
        self._captured = {}         # what captured steps work on, by identity: graphs may write to it after it has been replaced
        self._reset()
        self._device = None
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    def _reset(self):
        # parameter -> (arena, block0, a tensor without memory of the parameter's shape and order then, its state's tensors there)
        self._where = {}
        self._arenas = []
        self._plan = None
        self._known = None          # the states as the last plan found or made them (see _holds)

    def add_param_group(self, group):
        super().add_param_group(group)
        group = self.param_groups[-1]
        try:
            self._check_group(group)
        except Exception:
            self.param_groups.pop()
            raise
        self._plan = None

    def _check_group(self, group):
        device = self._device
        lr, (b1, b2) = group['lr'], group['betas']
        if isinstance(lr, torch.Tensor):
            if not self.capturable:
                raise ValueError('lr as a tensor needs an optimiser with capturable=True')
        elif not 0.0 <= lr:
            raise ValueError(f'Invalid learning rate: {lr}')
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f'Invalid betas: {group["betas"]}')
        if not 0.0 <= group['eps']:
            raise ValueError(f'Invalid epsilon value: {group["eps"]}')
        if not 0.0 <= group['weight_decay']:
            raise ValueError(f'Invalid weight_decay value: {group["weight_decay"]}')
        if bool(group.get('maximize', self.maximize)) != self.maximize:
            raise ValueError(f'a group with maximize={group["maximize"]}: all groups go the same way (an argument of the constructor)')
        if group.get('amsgrad'):
            raise ValueError('amsgrad is not supported')
        for p in group['params']:
            _check_tensor(p, 'a parameter')
            if not _dense(p):
                raise ValueError('a parameter is not dense (its elements do not fill one stretch of memory)')
            if self.master_weights and p.dtype == torch.float16:
                raise ValueError('master_weights keeps the low halves of bfloat16 parameters; float16 ones have none')
            if device is None:
                device = p.device
            elif p.device != device:
                raise ValueError(f'parameters on {device} and {p.device}')
        if len({id(p) for p in group['params']}) < len(group['params']):
            raise ValueError('a parameter appears twice')
        if isinstance(lr, torch.Tensor):
            _check_lr(lr, device)
        self._device = device

    # -- states ----------------------------------------------------------------------------------------------------------
    def _make_states(self, params):
        """states of parameters that have none, or have some from elsewhere (a loaded, copied or replaced state): one arena per
        type.  Nothing is changed unless all of them fit"""
        by_type, steps, to, source, made, arenas = {}, {}, [], [], [], []
        for p in params:
            by_type.setdefault(p.dtype, []).append(p)
        for dtype, ps in by_type.items():
            arena = _Arena(dtype, sum(-(-p.numel() // BLOCK) for p in ps), self.state_bits, self.master_weights, self._device)
            arenas.append(arena)
            block0 = 0
            for p in ps:
                mine, had = arena.views(p, block0), self.state.get(p)
                if had:
                    for name, view in mine.items():
                        if name not in had:
                            raise ValueError(f'the state of a parameter has no {name!r}: it comes from an optimiser with other '
                                             f'state_bits or master_weights (it has {sorted(map(str, had))})')
                        old = had[name]
                        if tuple(old.shape) != tuple(view.shape):
                            raise ValueError(f'state {name!r} has shape {tuple(old.shape)}, the parameter needs {tuple(view.shape)}')
                        to.append(view)
                        source.append(old)
                    if 'step' not in had:
                        raise ValueError("the state of a parameter has no 'step'")
                count = float(had['step']) if had else 0.0
                if count not in steps:
                    steps[count] = torch.tensor(count, dtype=torch.float32, device=self._device if self.capturable else 'cpu')
                made.append((p, {'step': steps[count], **mine}, (arena, block0, torch.empty_strided(p.shape, p.stride(), dtype=p.dtype, device='meta'),
                                                                 [(name, view, view.data_ptr()) for name, view in mine.items()])))
                block0 += -(-p.numel() // BLOCK)
        if to:
            with torch.no_grad():
                torch._foreach_copy_(to, source)
        self._arenas += arenas
        for p, state, where in made:
            self.state[p], self._where[p] = state, where

    # A program may replace what `state` holds: an entry, the state of a parameter, all of it.  The kernels work on the arenas, so
    # each step compares, and what is not the arena's any more is copied into a new one, as a loaded state is
    def _know(self):
        """notes the states as they are"""
        known, dicts, tensors = [], [], {}
        for p, state in self.state.items():
            where = self._where.get(p)
            if where is None:
                continue
            names = where[0].names
            known += (p, state)
            dicts.append(state)
            for item in state.items():
                if item[0] in names:
                    known += item
                    if isinstance(item[1], torch.Tensor):      # (a count that the program has set may be a number)
                        tensors[id(item[1])] = item[1]
            known.append(None)
        tensors = list(tensors.values())
        note, at = _words(1 + len(dicts) + 2 * len(tensors))
        _host().note(self.state, dicts, tensors, at)
        self._known = (known, dicts, tensors, at), note

    def _holds(self):
        return self._known is not None and _host().held(self.state, *self._known[0])

    def _sift(self):
        """parameters whose states are no longer where they were made lose their place"""
        self._plan = self._known = None
        for p, (_, _, _, views) in list(self._where.items()):
            st = self.state.get(p)
            if not (st and 'step' in st and all(st.get(name) is view and view.data_ptr() == at for name, view, at in views)):
                del self._where[p]

    def flat_state(self):
        """{name: [the flat buffers that hold this state]}: one per element type, the parameters' states one behind the other in
        the order of the parameter list, each from a multiple of 256 elements on ('..._scale': one value per 256).  States that
        were made in a later step, replaced by the program or brought into another memory order follow in buffers of their own; the
        place that such a state had before holds what was there"""
        out = {}
        for arena in self._arenas:
            for name, buf in arena.bufs.items():
                out.setdefault(name, []).append(buf)
        return out

    def __getstate__(self):
        keep = ('state_bits', 'master_weights', 'maximize', 'clip_norm', 'capturable', 'seed', '_device')
        return {**super().__getstate__(), **{k: getattr(self, k) for k in keep}}

    def __setstate__(self, state):
        super().__setstate__(state)
        self.grad_norm = None
        self.__dict__.setdefault('_captured', {})
        self._reset()

    def state_dict(self):
        # between the base class and the program's own hooks, which see what is returned
        hook = self.register_state_dict_post_hook(FusedAdamW._complete, prepend=True)
        try:
            return super().state_dict()
        finally:
            hook.remove()

    def _complete(self, sd):
        # here parameters that are stepped together share one count; another optimiser would count it once for each of them
        sd['state'] = {k: {**v, 'step': v['step'].clone()} if isinstance(v.get('step'), torch.Tensor) else v for k, v in sd['state'].items()}
        for g in sd['param_groups']:       # (where torch.optim.AdamW keeps it)
            g['maximize'] = self.maximize
        if self.state_bits == 8:           # whose blocks belong to stretches of memory, whatever the shape
            for k, p in enumerate(p for g in self.param_groups for p in g['params']):
                if 'step' in sd['state'].get(k, ()):
                    sd['state'][k]['order'] = _order(self._where[p][2] if p in self._where else p)

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        before = {k: self.__dict__[k] for k in ('state', 'param_groups', 'grad_norm', '_where', '_arenas', '_plan', '_known')}
        taken = {}

        def take(_, sd):                   # behind the program's own hooks, which may replace the dictionary
            groups = sd['param_groups']
            if any(g.get('amsgrad') for g in groups):
                raise ValueError('load_state_dict: amsgrad states are not supported')
            if any(bool(g.get('maximize', self.maximize)) != self.maximize for g in groups):
                raise ValueError(f'load_state_dict: maximize is {not self.maximize} in the dictionary and {self.maximize} here (a choice of the constructor)')
            taken.update(sd)
            # the base class would convert the states to their parameters' type: it gets the groups alone
            return {**sd, 'state': {}}

        def fill(_):                       # before the program's own hooks, which see the states
            ours, theirs = [p for g in self.param_groups for p in g['params']], [i for g in taken['param_groups'] for i in g['params']]
            saved = taken['state']
            self.state = defaultdict(dict, {p: dict(saved[i]) for i, p in zip(theirs, ours) if saved.get(i)})
            for p, st in self.state.items():
                if tuple(st.pop('order', _order(p))) != _order(p):
                    raise ValueError('load_state_dict: the 8-bit state of a parameter belongs to another memory order than it has')
            for g in self.param_groups:
                self._check_group(g)
            if self.state:                 # (groups without parameters have no device)
                with _lib.device_guard(self._device):
                    self._make_states(list(self.state))

        hooks = self.register_load_state_dict_pre_hook(take), self.register_load_state_dict_post_hook(fill, prepend=True)
        try:
            super().load_state_dict(state_dict)
        except Exception:                  # an optimiser that cannot take the dictionary is left as it was
            self.__dict__.update(before)
            raise
        finally:
            for hook in hooks:
                hook.remove()

    # -- the step --------------------------------------------------------------------------------------------------------
    def _build(self, capturing):
        """the launches of a step of the parameters that have gradients now"""
        every = [(g, p) for g in self.param_groups for p in g['params']]
        active = [(g, p, k) for k, (g, p) in enumerate(every) if p.grad is not None]
        if capturing:
            raise RuntimeError('FusedAdamW: the first step, and the first one with gradients for other parameters than before, cannot '
                               'be captured into a graph: take it eagerly')
        same = self._holds()
        if not same:
            self._sift()
        # (_gather asks this of every step; here it is asked before states are made)
        if _overlap([(p.data_ptr(), p.numel() * p.element_size()) for _, p, _ in active]):
            raise RuntimeError('FusedAdamW: two parameters share their memory')
        new = [p for _, p, _ in active if p not in self._where]
        if new:
            self._make_states(new)
        used = {id(where[0]) for where in self._where.values()}
        self._arenas = [a for a in self._arenas if id(a) in used]
        # a class: a group's parameters of one arena at the same step.  They share one count, which the call increments once.
        # On the device the values are unknown: there, what has shared a count so far goes on sharing it
        holders, classes, values, counts = {}, {}, {}, {}
        count_device = self._device if self.capturable else torch.device('cpu')
        if self.capturable and same:
            for p in self._where:
                step = self.state[p]['step']
                holders[id(step)] = holders.get(id(step), 0) + 1
        for g, p, k in active:
            (arena, block0, like, _), st = self._where[p], self.state[p]
            step = st['step']
            value = values.get(id(step))
            if value is None and not (isinstance(step, torch.Tensor) and step.dim() == 0 and step.dtype == torch.float32 and step.device == count_device):
                count = float(step)                # (put there by the program)
                if count not in counts:
                    counts[count] = torch.tensor(count, dtype=torch.float32, device=count_device)
                step = counts[count]
                value = values.get(id(step))
            if value is None:
                value = values[id(step)] = id(step) if self.capturable else float(step)
            key = (id(arena), id(g), value)
            if key not in classes:
                classes[key] = (arena, g, step, [])
            classes[key][3].append((p, block0, k, like, st))
        counted = {}
        for key, (arena, g, step, members) in classes.items():
            if holders.get(id(step)) != len(members):      # (the program may hold the count of a state that it has replaced)
                step = step.clone()
            for _, _, _, _, st in members:
                st['step'] = step
            counted[key] = step
        launches = []
        for arena in self._arenas:
            keys = [k for k in classes if k[0] == id(arena)]
            for at in range(0, len(keys), _CLASSES):
                part = keys[at:at + _CLASSES]
                members = sorted(((p, c, b, o, like) for c, key in enumerate(part) for p, b, o, like, _ in classes[key][3]), key=lambda m: m[3])
                launches.append(_Launch(arena, members, [(classes[key][1], counted[key]) for key in part]))
        self._plan = _Plan(launches, self.param_groups)
        self._know()
        return self._plan

    @torch.no_grad()
    def _gather_slowly(self, launch):
        """addresses of a launch whose tensors are not all plain: gradients of another memory order go through a copy (returned,
        to be kept until the launch is enqueued), a parameter that has got another order itself needs its state in that order,
        everything else that the kernels cannot take is an error"""
        kept = []
        if any(p.grad is None for p in launch.params):
            raise _Ungraded
        for k, p in enumerate(launch.params):
            g, dtype = p.grad, launch.arena.dtype
            if g.layout != torch.strided:
                raise RuntimeError('FusedAdamW does not support sparse gradients')
            if p.numel() != launch.sizes[k] or g.numel() != launch.sizes[k]:
                raise RuntimeError('FusedAdamW: a parameter has another size than its state')
            if p.device != self._device or g.device != self._device or p.dtype != dtype or g.dtype != dtype:
                raise RuntimeError(f'FusedAdamW: a parameter or gradient is no longer a {dtype} tensor on {self._device}')
            if not _dense(p) or p.is_neg():
                raise RuntimeError('FusedAdamW: a parameter is no longer dense')
            if not _same_order(p, launch.like[k]):
                raise _Reordered
            if g.is_neg() or not (_dense(g) and _same_order(p, g)):
                g = torch.empty_like(p).copy_(g)
                kept.append(g)
            launch.ptrs[k], launch.grads[k] = p.data_ptr(), g.data_ptr()
        return kept

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if self._device is None:                                # (groups without parameters)
            return loss
        with _lib.device_guard(self._device):
            capturing = torch.cuda.is_current_stream_capturing()
            if capturing and not self.capturable:
                raise RuntimeError('FusedAdamW: a step is captured into a graph only with capturable=True')
            plan = self._plan if self._plan is not None and self._fits(self._plan) else self._build(capturing)
            kept = None
            while kept is None:
                try:
                    kept = self._gather(plan)
                except _Ungraded:
                    plan = self._build(capturing)
                except _Reordered:
                    self._reorder()
                    plan = self._build(capturing)
            self._run(plan, capturing)
            del kept
        return loss

    def _gather(self, plan):
        """the addresses of a step, checked; returns what has to live until they are used"""
        kept, host = [], _host()
        for x in plan.launches:
            if host.gather(x.params, x.like, x.state.dtype, self._device.index, x.size_at, x.ptr_at, x.grad_at) != -1:
                kept += self._gather_slowly(x)
        # workgroups of one launch would read and write the same elements
        if host.overlap(plan.stretches):
            raise RuntimeError('FusedAdamW: two parameters share their memory')
        return kept

    def _reorder(self):
        """states of parameters whose memory has got another order: 32-bit ones move into it, 8-bit ones (blocks of memory) cannot"""
        if self.state_bits == 8:
            raise RuntimeError('FusedAdamW: a parameter has another memory order than its 8-bit state')
        for p in [p for p, (_, _, like, _) in self._where.items() if not _same_order(p, like)]:
            del self._where[p]

    def _fits(self, plan):
        return _host().fits(self.param_groups, plan.params, plan.mask, plan.groups) and self._holds()

    def _run(self, plan, capturing):
        device, L, host = self._device, _lib.lib(), _host()
        stream = _stream(device)
        rows, norm = None, None
        if self.clip_norm is not None:
            lists = [(x.state.dtype, x.grad_at, x.size_at, x.count) for x in plan.launches if x.total]
            if lists:
                rows = _norm_rows(lists, 2, device, stream)
                norm = torch.empty((), dtype=torch.float32, device=device)
            else:
                norm = torch.zeros((), dtype=torch.float32, device=device)
        self.grad_norm = norm
        for x in plan.launches:
            st = x.state
            st.bits, st.maximize, st.seed = self.state_bits, self.maximize, self.seed
            if rows is not None:
                st.norm_rows, st.norm_out, st.limit = rows.data_ptr(), norm.data_ptr(), _limit(self.clip_norm)
            else:
                st.norm_rows = None
            if self.capturable:
                hyper = torch.empty(_HYPER_BYTES, dtype=torch.uint8, device=device)
                st.hyper = hyper.data_ptr()
            for c, (g, step, count) in zip(x.table, x.classes):
                lr = g['lr']
                c.beta1, c.beta2 = g['betas']
                c.eps, c.weight_decay = g['eps'], g['weight_decay']
                if self.capturable:
                    c.step_dev = step.data_ptr()
                    if isinstance(lr, torch.Tensor):
                        _check_lr(lr, device)
                        c.lr_dev, c.lr = lr.data_ptr(), 0.0
                    else:
                        c.lr_dev, c.lr = None, lr
                else:
                    c.step, c.lr = int(count) + 1, lr
            rc = L.pdes_adamw_step(x.ptr_at, x.grad_at, x.tensor_at, x.count, x.table, len(x.classes), ctypes.byref(st), stream)
            _lib.check(rc, 'pdes_adamw_step')
            if not self.capturable:
                for _, _, count in x.classes:
                    count += 1
            host.changed(x.params, False)
            if capturing:
                self._captured.update((id(kept), kept) for kept in [x.arena] + [t for g, step, _ in x.classes for t in (step, g['lr'])])
            else:                           # what is replaced later is freed later than this stream's work on it
                if x.arena.stream != stream:
                    for buf in x.arena.bufs.values():
                        buf.record_stream(torch.cuda.current_stream(device))
                if self.capturable:
                    for _, step, count in x.classes:
                        if count is None:                           # (on the device)
                            step.record_stream(torch.cuda.current_stream(device))
