"""FusedAdamW's host side on CPU tensors: `host_only` takes its device checks away and computes the one C entry of a step
(pdes_adamw_step: fp32 parameters, 32-bit states, no clipping) in numpy, through the addresses that the call passes.  What the
optimiser decides on the host -- which states, counts and groups a step uses, what it refuses -- is what these tests see."""
import ctypes
import types

import numpy as np
import torch

BLOCK = 256


def _floats(address, n):
    return np.frombuffer((ctypes.c_float * n).from_address(address), dtype=np.float32) if n else np.zeros(0, np.float32)


class Entries:
    """stands in for the kernels' library"""

    def __init__(self):
        self.launches = []                   # tensors of each call

    def pdes_adamw_step(self, params, grads, tensors, count, classes, nclasses, state, stream):
        from pde_surrogate_amd.adamw import MtTensor
        st = state._obj
        assert st.dtype == 0 and st.bits == 32 and not st.norm_rows and 0 < nclasses <= 8
        p, g = ((ctypes.c_ulonglong * count).from_address(x) for x in (params, grads))
        t = (MtTensor * count).from_address(tensors)
        steps = []
        for c in classes[:nclasses]:
            if c.step_dev:
                _floats(c.step_dev, 1)[0] += 1
            steps.append(int(_floats(c.step_dev, 1)[0]) if c.step_dev else c.step)
        for k in range(count):
            n, c, step = t[k].n, classes[t[k].cls], steps[t[k].cls]
            assert t[k].block0 + -(-n // BLOCK) <= st.blocks
            w, grad = _floats(p[k], n), _floats(g[k], n) * (-1 if st.maximize else 1)
            m, v = (_floats(x + 4 * BLOCK * t[k].block0, n) for x in (st.exp_avg, st.exp_avg_sq))
            lr = _floats(c.lr_dev, 1)[0] if c.lr_dev else c.lr
            m[:] = c.beta1 * m + (1 - c.beta1) * grad
            v[:] = c.beta2 * v + (1 - c.beta2) * grad * grad
            w[:] = w * (1 - lr * c.weight_decay) - lr / (1 - c.beta1 ** step) * m / (np.sqrt(v) / np.sqrt(1 - c.beta2 ** step) + c.eps)
        self.launches.append(count)
        return 0


def host_only(monkeypatch):
    from pde_surrogate_amd import _lib, adamw
    entries, real = Entries(), adamw._host()
    # (every tensor takes the way of those that are not plain: gather accepts device tensors only)
    host = types.SimpleNamespace(**{k: getattr(real, k) for k in dir(real) if not k.startswith('_')})
    host.gather = lambda *a: 0
    monkeypatch.setattr(adamw, '_host', lambda: host)
    monkeypatch.setattr(adamw, '_check_tensor', lambda t, what: None)
    monkeypatch.setattr(adamw, '_stream', lambda device: 0)
    monkeypatch.setattr(_lib, 'lib', lambda: entries)
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: entries.capturing)
    entries.capturing = False
    return entries


def params(*sizes, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(n, generator=g)) for n in sizes]


def grads(ps, seed, which=None):
    g = torch.Generator().manual_seed(seed)
    for k, p in enumerate(ps):
        x = torch.randn(p.shape, generator=g)
        p.grad = x if which is None or k in which else None
