"""GPU tests of the list operators' arithmetic where lists are long, norms are not finite and roots are small."""
import math

import numpy as np
import pytest
import torch

import adamw_util as au

pytestmark = pytest.mark.gpu
DT = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}


@pytest.fixture(scope='module')
def dev():
    assert torch.cuda.is_available()
    return torch.device('cuda:0')


def _padding(buf, sizes):
    """which places of a flat buffer no element has"""
    free, at = torch.ones(buf.numel(), dtype=torch.bool, device=buf.device), 0
    for n in sizes:
        free[at:at + n] = False
        at += -(-n // au.BLOCK) * au.BLOCK
    return free


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('dtype,master', [('float32', False), ('bfloat16', False), ('bfloat16', True), ('float16', False)])
def test_a_norm_that_is_not_finite(dev, bits, dtype, master):
    """A finite clip_norm multiplies every gradient by min(1, clip_norm / (norm + 1e-6)), as torch.nn.utils.clip_grad_norm_ does: an
    infinite norm makes that 0 (and 0 * infinity NaN, in its own element alone), a NaN makes it NaN for every element.  What lies
    behind a tensor's last element stays zero"""
    from pde_surrogate_amd import optim
    sizes = [1, 255, 257, 1001, 2049]
    gen = torch.Generator().manual_seed(4)
    start = [(torch.randn(n, generator=gen) * 0.1).to(DT[dtype]).to(dev) for n in sizes]
    g = [torch.randn(n, generator=gen).to(DT[dtype]).to(dev) for n in sizes]
    for bad in (math.nan, math.inf, -math.inf):
        ps, qs = ([torch.nn.Parameter(x.clone()) for x in start] for _ in range(2))
        a, b = (optim.FusedAdamW(x, lr=1e-2, state_bits=bits, master_weights=master) for x in (ps, qs))
        for t in range(3):
            for k, (p, q) in enumerate(zip(ps, qs)):
                p.grad, q.grad = g[k] * (t + 1), g[k] * (t + 1)
                if t == 1:
                    q.grad.fill_(math.nan if math.isnan(bad) else 0.0)
                    if k == 3:
                        p.grad[0] = bad
                        q.grad[0] = math.nan
            a.clip_norm = 0.5 if t == 1 else None
            a.step()
            b.step()
            if t == 1:
                assert math.isnan(float(a.grad_norm)) if math.isnan(bad) else float(a.grad_norm) == math.inf
            for k, (p, q) in enumerate(zip(ps, qs)):
                spoilt = torch.full((sizes[k],), t > 0 and math.isnan(bad), device=dev)
                spoilt[0] = spoilt[0] or (t > 0 and k == 3)
                assert torch.equal(p.isnan(), spoilt) and torch.equal(q.isnan(), spoilt) and torch.equal(p[~spoilt], q[~spoilt]), (bad, t, k)
            for name, bufs in a.flat_state().items():
                if not name.endswith('_scale'):
                    assert not bufs[0].view(torch.uint8).view(bufs[0].numel(), -1)[_padding(bufs[0], sizes)].any(), (name, bad, t)
