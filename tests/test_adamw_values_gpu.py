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


@pytest.mark.parametrize('dtype,master', [('float32', False), ('bfloat16', False), ('bfloat16', True)])
def test_roots_of_very_small_second_moments(dev, dtype, master):
    """Gradients of 1e-18 to 1e-14, whose squares times 1e-3 are subnormal or a little above: the 8-bit states are their definition's, bit
    for bit, whatever their neighbours are (a lane works on eight elements at once, and roots of small numbers take another way)"""
    from pde_surrogate_amd import optim
    rng = np.random.default_rng(11)
    n = 256 * 3000
    mag = 10.0 ** rng.uniform(-18, -14, (n // 256, 1)) * np.exp(rng.uniform(-0.3, 0, (n // 256, 256)))     # (blocks of one size: their tops show)
    mag[::3, ::16] = 1e-21                                 # subnormal second moments among the others
    mag[1::3, ::32] = 0.0
    g = torch.from_numpy((mag * rng.choice([-1, 1], mag.shape)).astype(np.float32).reshape(-1)).to(DT[dtype]).to(dev)
    p = torch.nn.Parameter(torch.zeros(n, dtype=DT[dtype], device=dev))
    lr, betas, eps, wd, seed = 1e-3, (0.9, 0.999), 1e-8, 0.0, 3
    opt = optim.FusedAdamW([p], lr=lr, betas=betas, eps=eps, weight_decay=wd, state_bits=8, master_weights=master, seed=seed)
    blocks = n // 256
    q = [np.zeros((blocks, 256), np.float32), np.zeros(blocks, np.float32)] * 2
    for t in (1, 2):
        p.grad = g * t
        _, _, mc, ms, rc, rs = au.step8(np.zeros(n, np.float32), au.f64(p.grad).astype(np.float32), *q, t, lr, betas, eps, wd, seed, 0)
        opt.step()
        st = opt.state[p]
        for name, want in (('exp_avg_scale', ms), ('rms_scale', rs)):
            got = st[name].cpu().numpy()
            assert np.array_equal(got, want), f'{name}, step {t}: {int((got != want).sum())} of {blocks} differ'
        for name, want in (('exp_avg_q', mc), ('rms_q', rc)):
            got = st[name].view(torch.uint8).cpu().numpy().reshape(want.shape)
            assert np.array_equal(got, want), f'{name}, step {t}: {int((got != want).sum())} codes differ'
        q = [x for a in ('exp_avg', 'rms') for x in (st[a + '_q'].float().cpu().numpy().reshape(blocks, 256), st[a + '_scale'].cpu().numpy())]


@pytest.mark.parametrize('dtype,master', [('float32', False), ('bfloat16', False), ('bfloat16', True), ('float16', False)])
def test_roots_of_many_second_moments(dev, dtype, master):
    """Each of 2^18 blocks holds one element that is not zero, so that its scale is its root times 1 / 448: the scales of three steps are
    those of fp32 operations one by one"""
    from pde_surrogate_amd import optim
    blocks, b2 = 1 << 18, 0.999
    p = torch.nn.Parameter(torch.zeros(blocks * 256, dtype=DT[dtype], device=dev))
    p.grad = torch.zeros_like(p)
    gen = torch.Generator(dev).manual_seed(2)
    opt = optim.FusedAdamW([p], lr=0.0, betas=(0.9, b2), state_bits=8, master_weights=master, seed=1)
    r = np.zeros(blocks, np.float32)
    for t in range(1, 4):
        p.grad[::256] = torch.randn(blocks, generator=gen, device=dev).to(DT[dtype])
        opt.step()
        g = p.grad[::256].float().cpu().numpy()
        r = np.sqrt(r * r * np.float32(b2) + g * g * np.float32(1 - b2))
        want = r * np.float32(1 / 448)
        got = opt.state[p]['rms_scale'].cpu().numpy()
        assert want.dtype == np.float32 and np.array_equal(got, want), f'step {t}: {int((got != want).sum())} of {blocks} scales differ'
        r = opt.state[p]['rms_q'].view(blocks, 256)[:, 0].float().cpu().numpy() * got


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('dtype,master', [('float32', False), ('bfloat16', False), ('bfloat16', True), ('float16', False)])
def test_long_lists_step_as_short_ones(dev, bits, dtype, master):
    """34 M elements in one step, clipped: streaming accesses, the norm from a launch of its own, several tiles a workgroup where the rules
    say so.  The same tensors, a few at a time and not clipped, take none of these; with a clipping factor of exactly 1/2 and
    gradients halved by hand both do the same arithmetic, and their places in the list are the same: equal bits"""
    from pde_surrogate_amd import optim
    sizes = [1_000_003 + 517 * k for k in range(31)] + [1, 2048, 255, 3_100_000]
    assert sum(sizes) > 32 << 20
    gen = torch.Generator(dev).manual_seed(8)
    ps = [torch.nn.Parameter((torch.randn(n, generator=gen, device=dev) * 0.05).to(DT[dtype])) for n in sizes]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    a, b = (optim.FusedAdamW(x, lr=1e-2, weight_decay=0.1, state_bits=bits, master_weights=master, seed=6) for x in (ps, qs))
    few = [list(range(k, min(k + 4, len(ps)))) for k in range(0, len(ps), 4)]
    assert max(sum(sizes[k] for k in part) for part in few) < 6 << 20
    for t in range(2):
        g = [(torch.randn(n, generator=gen, device=dev) * 10.0 ** -(k % 3)).to(DT[dtype]) for k, n in enumerate(sizes)]
        for x in g:
            x[x.abs() < 2.0 ** -13] = 0                    # (halves of fp16's subnormal numbers would be rounded)
        g[33].zero_()                                      # brings the norm to 8192, so that the factor is 1 / 8192 * 4096
        left = 8192.0 ** 2 - sum(float(x.double().square().sum()) for x in g)
        for i in range(20):
            x = torch.tensor(math.sqrt(max(left, 0.0)) * (1 - 2.0 ** -8)).to(DT[dtype])
            if float(x) < 2.0 ** -13:
                break
            g[33][i] = x
            left -= float(x) ** 2
        assert 0 <= left < 8192.0 ** 2 * 2.0 ** -30
        for p, x in zip(ps, g):
            p.grad = x
        a.clip_norm = 4096.0
        a.step()
        assert float(a.grad_norm) == 8192.0 == float(optim.clip_grad_norm_(ps, math.inf))
        for part in few:
            for k, q in enumerate(qs):
                q.grad = g[k] * 0.5 if k in part else None
            b.step()
        for k, (p, q) in enumerate(zip(ps, qs)):
            assert torch.equal(p, q), (k, t)
            assert float(a.state[p]['step']) == float(b.state[q]['step']) == t + 1
            for name in a.state[p]:
                if name != 'step':
                    assert torch.equal(a.state[p][name].view(torch.uint8), b.state[q][name].view(torch.uint8)), (name, k, t)


@pytest.mark.parametrize('inside', [False, True])
def test_limits_beyond_fp32(dev, inside):
    """a limit that fp32 does not hold is a limit all the same: only infinity means none.  With an infinite norm the factor is 0"""
    from pde_surrogate_amd import optim
    for limit, factor in ((1e39, 0.0), (1e300, 0.0), (math.inf, 1.0)):
        ps = [torch.nn.Parameter(torch.zeros(5, device=dev)) for _ in range(2)]
        for p in ps:
            p.grad = torch.ones_like(p)
        ps[1].grad[2] = math.inf
        if inside:
            opt = optim.FusedAdamW(ps, lr=1.0, weight_decay=0.0, clip_norm=limit)
            opt.step()
            got, norm = opt.state[ps[0]]['exp_avg'] / np.float32(1 - 0.9), opt.grad_norm
        else:
            norm = optim.clip_grad_norm_(ps, limit)
            got = ps[0].grad
        assert float(norm) == math.inf and (got == factor).all()
    ps[1].grad[2] = 1.0
    ps[0].grad.fill_(1.0)
    assert float(optim.clip_grad_norm_(ps, 1e39)) == np.float32(math.sqrt(10)) and (ps[0].grad == 1).all()


@pytest.mark.parametrize('dtype', ['bfloat16', 'float16'])
def test_8_bit_states_of_16_bit_weights_are_their_definition(dev, dtype):
    """codes and scales bit for bit, as for fp32 weights (the weights themselves: one rounding of 16 bits, test_adamw_gpu.py)"""
    from pde_surrogate_amd import optim
    sizes = [1_500_007, 255, 1, 8192, 300_000]
    gen = torch.Generator().manual_seed(17)
    ps = [torch.nn.Parameter((torch.randn(n, generator=gen) * 0.05).to(DT[dtype]).to(dev)) for n in sizes]
    lr, betas, eps, wd, seed = 2e-3, (0.9, 0.95), 1e-8, 0.1, 5
    opt = optim.FusedAdamW(ps, lr=lr, betas=betas, eps=eps, weight_decay=wd, state_bits=8, seed=seed)
    for t in range(1, 4):
        before = []
        for k, p in enumerate(ps):
            p.grad = (torch.randn(sizes[k], generator=gen) * 10.0 ** -k).to(DT[dtype]).to(dev)
            st, blocks = opt.state.get(p, {}), -(-sizes[k] // au.BLOCK)
            before.append([x for a in ('exp_avg', 'rms') for x in (
                (st[a + '_q'].float().cpu().numpy().reshape(blocks, au.BLOCK), st[a + '_scale'].cpu().numpy()) if st
                else (np.zeros((blocks, au.BLOCK), np.float32), np.zeros(blocks, np.float32)))])
        opt.step()
        for k, p in enumerate(ps):
            _, _, mc, ms, rc, rs = au.step8(np.zeros(sizes[k], np.float32), au.f64(p.grad).astype(np.float32), *before[k], t, lr, betas, eps, wd, seed, k)
            st = opt.state[p]
            for name, want in (('exp_avg_q', mc), ('rms_q', rc)):
                got = st[name].view(torch.uint8).cpu().numpy().reshape(want.shape)
                assert np.array_equal(got, want), f'{name} of tensor {k}, step {t}: {int((got != want).sum())} codes differ'
            assert np.array_equal(st['exp_avg_scale'].cpu().numpy(), ms) and np.array_equal(st['rms_scale'].cpu().numpy(), rs), (k, t)
