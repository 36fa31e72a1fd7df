"""GPU tests of the AdamW step over many tensors and of gradient clipping (pde_surrogate_amd/adamw.py, csrc/multi_tensor.hip)
against plain computations in 64 bits with derived bounds, and of the 8-bit states against their definition: bit for bit where fp32
weights are held (fp32, or bf16 with low halves)."""
import contextlib
import copy
import io
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


def _params(dev, sizes, dtype='float32', scale=0.05, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter((torch.randn(n, generator=g) * scale).to(DT[dtype]).to(dev)) for n in sizes]


def _grads(params, seed, spread=True):
    g = torch.Generator().manual_seed(seed)
    for k, p in enumerate(params):
        s = 10.0 ** (-(k % 4)) if spread else 1.0
        p.grad = (torch.randn(p.shape, generator=g) * s).to(p.dtype).to(p.device)



# ---- 32-bit states --------------------------------------------------------------------------------------------------------
SIZES = {
    'one': [1],
    'edges': [255, 256, 257, 3, 2047, 2048, 2049, 1, 0, 5],
    'many': [(37 * k) % 701 + 1 for k in range(230)],
    'long': [1_500_007, 13],
    'chunks': [9_000_001, 8192, 8191],
}


@pytest.mark.parametrize('sizes', sorted(SIZES))
@pytest.mark.parametrize('dtype,master', [('float32', False), ('bfloat16', False), ('bfloat16', True), ('float16', False)])
def test_step_with_32_bit_states_against_64_bits(dev, sizes, dtype, master):
    from pde_surrogate_amd import optim
    ps = _params(dev, SIZES[sizes], dtype)
    lr, betas, eps, wd = 2e-3, (0.9, 0.99), 1e-8, 0.1
    half = len(ps) // 2
    groups = [{'params': ps[:half], 'weight_decay': 0.0, 'lr': 5e-4}, {'params': ps[half:]}] if half else ps
    opt = optim.FusedAdamW(groups, lr=lr, betas=betas, eps=eps, weight_decay=wd, master_weights=master)
    for t in range(1, 4):
        _grads(ps, 10 + t)
        kept = [p.grad.clone() for p in ps]
        before = []
        for p in ps:
            st = opt.state.get(p, {})
            w = au.master64(p, st['low']) if master and t > 1 else au.f64(p)
            before.append((w, au.f64(st['exp_avg']) if st else np.zeros(p.numel()), au.f64(st['exp_avg_sq']) if st else np.zeros(p.numel())))
        opt.step()
        for k, (p, (w, m, v)) in enumerate(zip(ps, before)):
            a, b = (5e-4, 0.0) if half and k < half else (lr, wd)
            want, bound = au.step64(w, au.f64(kept[k]), m, v, t, a, betas, eps, b)
            st = opt.state[p]
            what = f'tensor {k} of {p.numel()}, step {t}'
            au.within(st['exp_avg'], want[1], bound[1], 'exp_avg of ' + what)
            au.within(st['exp_avg_sq'], want[2], bound[2], 'exp_avg_sq of ' + what)
            if master:
                full = au.master64(p, st['low'])
                au.within(full, want[0], bound[0], 'weight of ' + what)
                au.within(p, full, np.abs(full) * 2.0 ** -8 + 2.0 ** -134, 'upper half of ' + what)
            else:
                rounding = au.HALF[dtype] * (np.abs(want[0]) + bound[0]) + (2.0 ** -25 if dtype == 'float16' else 0)
                au.within(p, want[0], bound[0] + rounding, 'weight of ' + what)
            assert float(st['step']) == t
            assert torch.equal(p.grad, kept[k])
    for buf in opt.flat_state()['exp_avg']:          # what lies behind a tensor's last element stays zero
        used = torch.zeros_like(buf, dtype=torch.bool)
        at = 0
        for p in ps:
            used[at:at + p.numel()] = True
            at += -(-p.numel() // au.BLOCK) * au.BLOCK
        assert not buf[~used].any()


def test_step_equals_torch_adamw_in_use(dev):
    """DenseED training steps with clipping: the same gradients to torch.optim.AdamW (clipped by torch) on copies"""
    from pde_surrogate_amd import optim
    from pde_surrogate_amd.models.codec import DenseED
    from pde_surrogate_amd.models.darcy import conv_boundary_condition, conv_constitutive_constraint, conv_continuity_constraint
    from pde_surrogate_amd.utils.image_gradient import SobelFilter
    torch.manual_seed(1)
    with contextlib.redirect_stdout(io.StringIO()):
        net = DenseED(1, 3, 64, [3, 4, 3]).to(dev)
    sobel = SobelFilter(64, correct=True, device=dev)
    opt = optim.FusedAdamW(net.parameters(), lr=1e-3, weight_decay=0.05, clip_norm=0.5)
    copies, other = None, None
    for t in range(1, 5):
        x = torch.exp(0.3 * torch.randn(8, 1, 64, 64, device=dev))
        net.zero_grad()
        y = net(x)
        d, n = conv_boundary_condition(y)
        (conv_constitutive_constraint(x, y, sobel) + conv_continuity_constraint(y, sobel) + 10 * (d + n)).backward()
        ps = list(net.parameters())
        copies = [torch.nn.Parameter(p.detach().clone()) for p in ps]
        for c, p in zip(copies, ps):
            c.grad = p.grad.detach().clone()
        other = torch.optim.AdamW(copies, lr=1e-3, weight_decay=0.05)
        if t > 1:
            other.load_state_dict(copy.deepcopy(opt.state_dict()))     # (torch takes tensors of its own type as they are)
        norm = torch.nn.utils.clip_grad_norm_(copies, 0.5)
        opt.step()
        other.step()
        # torch's norm is an fp32 sum of fp32 norms: n_terms / 2 roundings at most, far under 1e-5 with its tree sums
        assert abs(float(opt.grad_norm) / float(norm) - 1) < 1e-5 and float(norm) > 0.5
        for p, c in zip(ps, copies):
            # both round each operation to fp32; the norms' difference moves g by 1e-5, an update by as much of lr at most
            assert float((p - c).detach().abs().max()) <= 4e-5 * 1e-3 * 40 + 2.0 ** -22 * float(c.detach().abs().max())


# ---- 8-bit states ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('sizes', ['one', 'edges', 'many', 'long', 'chunks'])
@pytest.mark.parametrize('dtype,master', [('float32', False), ('bfloat16', False), ('bfloat16', True), ('float16', False)])
def test_step_with_8_bit_states_is_its_definition(dev, sizes, dtype, master):
    from pde_surrogate_amd import optim
    ps = _params(dev, SIZES[sizes], dtype)
    lr, betas, eps, wd, seed = 2e-3, (0.9, 0.999), 1e-8, 0.1, 77
    opt = optim.FusedAdamW(ps, lr=lr, betas=betas, eps=eps, weight_decay=wd, state_bits=8, master_weights=master, seed=seed)
    for t in range(1, 4):
        _grads(ps, 20 + t)
        if t == 2:
            for p in ps[::2]:
                p.grad.zero_()
        before = []
        for p in ps:
            st = opt.state.get(p, {})
            n, blocks = p.numel(), -(-p.numel() // au.BLOCK)
            w = au.master64(p, st['low']) if master and t > 1 else au.f64(p)
            q = [(st[a + '_q'].float().cpu().numpy().reshape(blocks, au.BLOCK), st[a + '_scale'].cpu().numpy()) if st
                 else (np.zeros((blocks, au.BLOCK), np.float32), np.zeros(blocks, np.float32)) for a in ('exp_avg', 'rms')]
            before.append((w.astype(np.float32), au.f64(p.grad).astype(np.float32), *q[0], *q[1]))
        opt.step()
        for k, (p, b) in enumerate(zip(ps, before)):
            if not p.numel():
                continue
            w, size, mc, ms, rc, rs = au.step8(*b, t, lr, betas, eps, wd, seed, k)
            st, what = opt.state[p], f'tensor {k} of {p.numel()}, step {t}'
            codes = [(name, st[name].view(torch.uint8).cpu().numpy().reshape(want.shape), want) for name, want in (('exp_avg_q', mc), ('rms_q', rc))]
            scales = [(st[name].cpu().numpy().astype(np.float64), want.astype(np.float64)) for name, want in (('exp_avg_scale', ms), ('rms_scale', rs))]
            w = w.astype(np.float64)
            if master or dtype == 'float32':
                for name, got, want in codes:
                    assert np.array_equal(got, want), f'{name} of {what}: {int((got != want).sum())} codes differ'
                assert all(np.array_equal(x, y) for x, y in scales), what
                assert np.array_equal(au.master64(p, st['low']) if master else au.f64(p), w), f'weight of {what}'
            else:
                # weights of 16 bits: r may be the neighbouring number (2 u; its scale 4 u after its own rounding).  The change: the
                # denominator 3 u besides, the reciprocal 2 u, products and the definition's own roundings 5 u: under 20 u of the terms'
                # size.  The weight: 2 u, then its type's rounding
                assert np.array_equal(codes[0][1], codes[0][2]) and np.array_equal(*scales[0]), what
                au.codes_near(codes[1][1], codes[1][2], f'rms_q of {what}')
                assert np.all(np.abs(scales[1][0] - scales[1][1]) <= 4 * au.U * scales[1][1]), what
                bound = 20 * au.U * size.astype(np.float64) + (2 * au.U + au.HALF[dtype]) * np.abs(w) * (1 + 2.0 ** -20) + \
                    (2.0 ** -25 if dtype == 'float16' else au.TINY)
                au.within(p, w, bound, f'weight of {what}')


def test_8_bit_states_follow_the_moments_on_average(dev):
    """Constant gradients: m and v approach g and g^2 like the 32-bit moments.  Held with stochastic rounding (spacing 1/8 of
    the value at most) an element's r walks; its mean over many elements must not drift: 2048 equal elements, standard error of
    the mean of r under 0.25 / sqrt(2048) = 0.6 %, and 200 steps of beta2 = 0.99 move v to 1 - 0.99^200 = 0.866 of g^2"""
    from pde_surrogate_amd import optim
    p = torch.nn.Parameter(torch.zeros(2048, device=dev))
    opt = optim.FusedAdamW([p], lr=1e-3, betas=(0.9, 0.99), weight_decay=0.0, state_bits=8)
    p.grad = torch.full_like(p, 0.3)
    p.grad[::256] = 1.7                                  # a larger element in each block: the others do not sit at the top code
    for _ in range(200):
        opt.step()
    st = opt.state[p]
    r = st['rms_q'].float() * st['rms_scale'].repeat_interleave(256)
    m = st['exp_avg_q'].float() * st['exp_avg_scale'].repeat_interleave(256)
    plain = torch.arange(2048, device=dev) % 256 != 0
    # r^2 averages to v (the rounding of r adds a variance of spacing^2 / 4 at most a step, damped by beta2): 3 % is 5 deviations
    assert abs(float((r[plain] ** 2).mean()) / (0.09 * (1 - 0.99 ** 200)) - 1) < 0.06
    assert abs(float(m[plain].mean()) / 0.3 - 1) < 0.03


@pytest.mark.parametrize('bits', [32, 8])
def test_gradients_that_are_not_finite_spoil_their_own_elements_only(dev, bits):
    from pde_surrogate_amd import optim
    ps, qs = _params(dev, [1000, 300]), _params(dev, [1000, 300])
    bad = [(0, 5, math.nan), (0, 300, math.inf), (1, 299, -math.inf)]
    a, b = (optim.FusedAdamW(x, lr=1e-2, state_bits=bits) for x in (ps, qs))
    clean = [torch.ones(1000, dtype=torch.bool, device=dev), torch.ones(300, dtype=torch.bool, device=dev)]
    for t in range(3):
        _grads(ps, t)
        _grads(qs, t)
        for k, i, x in bad:
            clean[k][i] = False
            qs[k].grad[i] = 0.0
            if t == 1:
                ps[k].grad[i] = x
            else:
                ps[k].grad[i] = 0.0
        a.step()
        b.step()
    for k in range(2):
        assert torch.equal(ps[k][clean[k]], qs[k][clean[k]])
        assert not torch.isfinite(ps[k][~clean[k]]).any()


@pytest.mark.parametrize('dtype', sorted(DT))
def test_8_bit_states_without_eps(dev, dtype):
    """eps = 0 counts as 2^-100: zeros stay zeros (where 32-bit states give 0 / 0), and a gradient whose square vanishes in fp32 steps by
    lr g 2^100.  In general by lr m / (r / sqrt(1 - beta2) + 2^-100) / (1 - beta1), m and r from fp32 products; the parameter's type
    rounds that by 2^-8 at most, subnormal operands lose up to 2^-4 of themselves before (g = 1e-44 has three bits)"""
    from pde_surrogate_amd import optim
    f = np.float32
    g = torch.tensor([0.0, 1e-7, 6e-5, 1e-3, 1.0] if dtype == 'float16' else [0.0, 1e-44, 1e-38, 1e-30, 1e-23, 1e-15, 1.0]).to(DT[dtype]).to(dev)
    for k in range(g.numel()):
        p = torch.nn.Parameter(torch.zeros(300, device=dev, dtype=DT[dtype]))
        opt = optim.FusedAdamW([p], lr=1e-2, eps=0.0, weight_decay=0.0, state_bits=8)
        p.grad = torch.zeros_like(p)
        p.grad[7] = g[k]
        opt.step()
        x = f(float(g[k]))
        r = np.sqrt(x * x * f(1 - 0.999))
        want = 1e-2 * float(x * f(1 - 0.9)) / 0.1 / (float(r) / math.sqrt(1 - 0.999) + 2.0 ** -100)
        got = p.detach().float()
        assert torch.isfinite(got).all() and not got[:7].any() and not got[8:].any()
        assert abs(float(got[7]) + want) <= want * (2.0 ** -8 + (2.0 ** -4 if 0 < float(x) < 1e-37 else 1e-6)), (float(x), float(got[7]), want)


@pytest.mark.parametrize('bits', [32, 8])
def test_zero_and_tiny_gradients(dev, bits):
    """m = v = 0 gives 0 / eps = 0: only the decay moves the weight; gradients whose squares vanish in fp32 stay harmless"""
    from pde_surrogate_amd import optim
    ps = _params(dev, [513, 513])
    start = [p.detach().clone() for p in ps]
    opt = optim.FusedAdamW(ps, lr=1e-2, weight_decay=0.5, state_bits=bits)
    for _ in range(2):
        ps[0].grad, ps[1].grad = torch.zeros_like(ps[0]), torch.full_like(ps[1], 1e-30)
        opt.step()
    f = np.float32(1 - 1e-2 * 0.5)
    assert np.array_equal(ps[0].detach().cpu().numpy(), start[0].cpu().numpy() * f * f)
    # m / (0 + eps) = 1e-30 / 1e-8: a change of 1e-24
    assert float((ps[1].detach() - start[1] * float(f) ** 2).abs().max()) < 1e-7


# ---- clipping -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('sizes', sorted(SIZES))
@pytest.mark.parametrize('dtype', sorted(DT))
@pytest.mark.parametrize('kind', [2.0, math.inf])
def test_clip_grad_norm(dev, sizes, dtype, kind):
    from pde_surrogate_amd import optim
    ps = _params(dev, SIZES[sizes], dtype)
    _grads(ps, 3)
    before = [au.f64(p.grad) for p in ps]
    every = np.concatenate(before)
    norm = np.sqrt((every ** 2).sum()) if kind == 2.0 else np.abs(every).max()
    # fp64 sums of exact squares: the result is rounded to fp32 once (and its fp64 roundings, which do not count)
    got = optim.clip_grad_norm_(ps, math.inf, kind)
    assert got.dtype == torch.float32 and got.shape == () and abs(float(got) - norm) <= 1.001 * au.U * norm
    got = optim.clip_grad_norm_(ps, float(norm) * 1.5, kind)                      # under the limit: not a bit changes
    assert all(np.array_equal(au.f64(p.grad), b) for p, b in zip(ps, before))
    limit = float(norm) * 0.25
    got = optim.clip_grad_norm_(ps, limit, kind)
    assert abs(float(got) - norm) <= 1.001 * au.U * norm
    factor = limit / (norm + 1e-6)
    for p, b in zip(ps, before):
        # the factor: norm, its sum, the reciprocal, the product and the limit round to fp32; the product with g; g's type
        bound = np.abs(b * factor) * (6 * au.U + au.HALF[dtype] * (1 + 6 * au.U)) + (2.0 ** -25 if dtype == 'float16' else au.TINY)
        au.within(p.grad, b * factor, bound, 'clipped gradient')


def test_clip_grad_norm_of_mixed_types_and_values(dev):
    from pde_surrogate_amd import optim
    ps = _params(dev, [1000, 77], 'float32') + _params(dev, [513], 'bfloat16') + _params(dev, [300, 1], 'float16')
    _grads(ps, 5, spread=False)
    ps.append(torch.nn.Parameter(torch.zeros(5, device=dev)))                      # without a gradient
    want = math.sqrt(sum(float((au.f64(p.grad) ** 2).sum()) for p in ps if p.grad is not None))
    assert abs(float(optim.clip_grad_norm_(iter(ps), math.inf)) / want - 1) <= 1.001 * au.U
    optim.clip_grad_norm_(ps, want / 3)
    assert abs(float(optim.clip_grad_norm_(ps, math.inf)) / (want / 3) - 1) < 2.0 ** -8
    # huge and tiny values: their squares leave fp32's range, the norm does not
    big = [torch.nn.Parameter(torch.zeros(7, device=dev)) for _ in range(2)]
    big[0].grad, big[1].grad = torch.full((7,), 3e30, device=dev), torch.full((7,), -4e30, device=dev)
    assert abs(float(optim.clip_grad_norm_(big, math.inf)) / (5e30 * math.sqrt(7)) - 1) < 4 * au.U
    big[0].grad, big[1].grad = torch.full((7,), 3e-30, device=dev), torch.full((7,), -4e-30, device=dev)
    assert abs(float(optim.clip_grad_norm_(big, math.inf)) / (5e-30 * math.sqrt(7)) - 1) < 4 * au.U
    # zeros; NaN and infinity, in either norm; error_if_nonfinite leaves everything as it was
    big[0].grad, big[1].grad = torch.zeros(7, device=dev), torch.zeros(7, device=dev)
    assert float(optim.clip_grad_norm_(big, 1.0)) == 0.0 and not big[0].grad.any()
    for x in (math.nan, math.inf):
        for kind in (2.0, math.inf):
            big[0].grad, big[1].grad = torch.ones(7, device=dev), torch.ones(7, device=dev)
            big[1].grad[3] = x
            got = float(optim.clip_grad_norm_(big, math.inf, kind))
            assert math.isnan(got) if math.isnan(x) else got == math.inf
            assert torch.equal(big[0].grad, torch.ones(7, device=dev))
            with pytest.raises(RuntimeError, match='not finite'):
                optim.clip_grad_norm_(big, 1.0, kind, error_if_nonfinite=True)
            assert torch.equal(big[0].grad, torch.ones(7, device=dev))
    got = optim.clip_grad_norm_(big, 0.0)                                           # infinity: the factor is 0, as in torch
    assert float(got) == math.inf and not big[0].grad.any() and math.isnan(float(big[1].grad[3]))
    big[0].grad, big[1].grad = torch.ones(7, device=dev), torch.ones(7, device=dev)
    assert float(optim.clip_grad_norm_(big, 2.0, error_if_nonfinite=True)) == pytest.approx(math.sqrt(14), rel=2e-7)
    assert float(big[0].grad[0]) == pytest.approx(2 / math.sqrt(14), rel=1e-6)
    assert float(optim.clip_grad_norm_([], 1.0)) == 0.0


@pytest.mark.parametrize('bits,dtype,master', [(32, 'float32', False), (32, 'bfloat16', True), (8, 'float32', False), (8, 'bfloat16', True)])
@pytest.mark.parametrize('maximize', [False, True])
def test_step_with_clipping_equals_clipping_then_step(dev, bits, dtype, master, maximize):
    """clip_norm multiplies the gradients as they are read: what the step does to gradients that a plain product with the same
    factor has clipped in fp32.  `.grad` stays, grad_norm is the norm; groups, types and launches share one norm"""
    from pde_surrogate_amd import optim
    sizes = SIZES['many']
    kw = dict(lr=1e-3, state_bits=bits, master_weights=master, maximize=maximize, seed=5)
    ps, qs = _params(dev, sizes, dtype), _params(dev, sizes, 'float32')
    for p, q in zip(ps, qs):
        q.data.copy_(p.data)
    a = optim.FusedAdamW([{'params': ps[:100]}, {'params': ps[100:], 'weight_decay': 0.0}], clip_norm=0.7, **kw)
    b = optim.FusedAdamW([{'params': qs[:100]}, {'params': qs[100:], 'weight_decay': 0.0}], **dict(kw, master_weights=False))
    for t in range(3):
        _grads(ps, t)
        kept = [p.grad.clone() for p in ps]
        norm = math.sqrt(sum(float((au.f64(p.grad) ** 2).sum()) for p in ps))
        a.step()
        assert abs(float(a.grad_norm) - norm) <= 1.001 * au.U * norm
        f = np.float32(1) / (a.grad_norm.cpu().numpy() + np.float32(1e-6)) * np.float32(0.7)
        for p, q, g in zip(ps, qs, kept):
            assert torch.equal(p.grad, g)
            q.grad = g.float() * float(f)
        b.step()
        for p, q in zip(ps, qs):
            if master:
                assert np.array_equal(au.master64(p, a.state[p]['low']), au.f64(q))
            else:
                assert torch.equal(p, q)
            for k in a.state[p]:
                if k not in ('low', 'step'):
                    assert torch.equal(a.state[p][k].view(torch.uint8), b.state[q][k].view(torch.uint8)), k


# ---- memory: views, alignment, orders, neighbours -----------------------------------------------------------------------
@pytest.mark.parametrize('dtype', sorted(DT))
@pytest.mark.parametrize('bits', [32, 8])
def test_views_at_any_offset_and_their_neighbours(dev, dtype, bits):
    from pde_surrogate_amd import optim
    sizes = [1, 7, 256, 1001, 4099, 20003]
    flat = torch.full((sum(sizes) + 50,), 9.0, device=dev, dtype=DT[dtype])
    gflat = torch.full_like(flat, 7.0)
    gen = torch.Generator().manual_seed(3)
    ps, alone, at, free = [], [], 3, torch.ones(flat.numel(), dtype=torch.bool, device=dev)
    for n in sizes:
        x, g = torch.randn(n, generator=gen).to(DT[dtype]).to(dev), torch.randn(n, generator=gen).to(DT[dtype]).to(dev)
        flat[at:at + n], gflat[at + 1:at + 1 + n] = x, g
        free[at:at + n] = False
        ps.append(torch.nn.Parameter(flat[at:at + n]))
        ps[-1].grad = gflat[at + 1:at + 1 + n]
        alone.append(torch.nn.Parameter(x.clone()))
        alone[-1].grad = g.clone()
        at += n + 5
    gkeep = gflat.clone()
    a, b = (optim.FusedAdamW(x, lr=1e-2, state_bits=bits, clip_norm=1.0) for x in (ps, alone))
    for _ in range(2):
        a.step()
        b.step()
    for p, q in zip(ps, alone):
        assert p.data_ptr() >= flat.data_ptr() and torch.equal(p, q)
    assert (flat[free] == 9.0).all() and torch.equal(gflat, gkeep)
    c, d = optim.clip_grad_norm_(ps, 0.1), optim.clip_grad_norm_(alone, 0.1)
    assert torch.equal(c, d)
    for p, q in zip(ps, alone):
        assert torch.equal(p.grad, q.grad)
        gkeep[(p.grad.data_ptr() - gflat.data_ptr()) // flat.element_size():][:p.numel()] = p.grad
    assert torch.equal(gflat, gkeep)


def test_memory_orders(dev):
    """channels-last and transposed parameters, gradients of another order, an expanded gradient"""
    from pde_surrogate_amd import optim
    torch.manual_seed(0)
    w = [torch.randn(8, 6, 3, 3, device=dev), torch.randn(40, 30, device=dev), torch.randn(33, 17, device=dev), torch.randn(5, 4, device=dev)]
    g = [torch.randn(8, 6, 3, 3, device=dev), torch.randn(40, 30, device=dev), torch.randn(33, 17, device=dev), torch.ones(5, 4, device=dev)]
    ps = [torch.nn.Parameter(w[0].to(memory_format=torch.channels_last)), torch.nn.Parameter(w[1].t().contiguous().t()),
          torch.nn.Parameter(w[2].clone()), torch.nn.Parameter(w[3].clone())]
    ps[0].grad, ps[1].grad = g[0].clone(), g[1].clone()
    ps[2].grad = g[2].t().contiguous().t()
    ps[3].grad = torch.ones(1, 1, device=dev).expand(5, 4)
    qs = [torch.nn.Parameter(x.clone()) for x in w]
    for q, x in zip(qs, g):
        q.grad = x.clone()
    a, b = optim.FusedAdamW(ps, lr=1e-2), optim.FusedAdamW(qs, lr=1e-2)
    for _ in range(2):
        a.step()
        b.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q) and torch.equal(a.state[p]['exp_avg'], b.state[q]['exp_avg'])
        assert a.state[p]['exp_avg'].stride() == p.stride()
    with pytest.raises(RuntimeError, match='not dense'):
        optim.clip_grad_norm_(ps, 1.0)
    norm, want = optim.clip_grad_norm_(ps[:3], 1.0), optim.clip_grad_norm_(qs[:3], 1.0)
    assert abs(float(norm) / float(want) - 1) <= 2.1 * au.U           # (summed in other orders in fp64, rounded once)
    for p, q in zip(ps[:3], qs[:3]):
        assert float((p.grad - q.grad).abs().max()) <= 1e-6


@pytest.mark.parametrize('dtype,master', [('float32', False), ('bfloat16', True)])
def test_a_parameter_whose_memory_order_changes(dev, dtype, master):
    """model.to(memory_format=channels_last) between steps: 32-bit states follow, 8-bit ones refuse"""
    from pde_surrogate_amd import optim
    torch.manual_seed(0)
    ps = [torch.nn.Parameter(torch.randn(8, 6, 3, 3, device=dev, dtype=DT[dtype])), torch.nn.Parameter(torch.randn(77, device=dev, dtype=DT[dtype]))]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    a, b = (optim.FusedAdamW(x, lr=1e-2, master_weights=master) for x in (ps, qs))
    c = optim.FusedAdamW([torch.nn.Parameter(ps[0].detach().clone())], state_bits=8)
    for t in range(4):
        _grads(qs, t)
        if t == 2:
            for x in (ps, c.param_groups[0]['params']):
                x[0].grad = None
                x[0].data = x[0].data.to(memory_format=torch.channels_last)
        for p, q in zip(ps, qs):
            p.grad = q.grad.clone(memory_format=torch.preserve_format) if t != 3 else q.grad.to(memory_format=torch.channels_last if q.dim() == 4 else torch.preserve_format)
        a.step()
        b.step()
        for p, q in zip(ps, qs):
            assert torch.equal(p, q) and float(a.state[p]['step']) == t + 1
            assert all(torch.equal(a.state[p][k], b.state[q][k]) for k in a.state[p])
        c.param_groups[0]['params'][0].grad = qs[0].grad.clone()
        if t < 2:
            c.step()
        else:
            with pytest.raises(RuntimeError, match='memory order'):
                c.step()
    assert a.state[ps[0]]['exp_avg'].stride() == ps[0].stride()


def test_a_group_whose_parameters_are_exchanged(dev):
    from pde_surrogate_amd import optim
    ps = _params(dev, [10, 20])
    _grads(ps, 0)
    opt = optim.FusedAdamW(ps[:1], lr=1e-2)
    opt.step()
    keep, other = ps[0].detach().clone(), ps[1].detach().clone()
    opt.param_groups[0]['params'][0] = ps[1]
    opt.step()
    assert torch.equal(ps[0], keep) and not torch.equal(ps[1], other) and float(opt.state[ps[1]]['step']) == 1


def test_overwritten_master_weights_are_taken_as_they_are(dev):
    """the program overwrites bf16 parameters (a loaded model, a pruned weight): the kept low half moves the weight by half a
    step at most, never across zero or into infinity"""
    from pde_surrogate_amd import optim
    p = _params(dev, [4096], 'bfloat16')[0]
    opt = optim.FusedAdamW([p], lr=1e-2, weight_decay=0.0, master_weights=True)
    p.grad = torch.randn_like(p)
    opt.step()
    low = opt.state[p]['low']
    assert (low < 0).any() and (low > 0).any()
    new = torch.randn(4096, device=dev).bfloat16()
    new[::4], new[1::8], new[2::8], new[3::16] = 0.0, -0.0, math.inf, math.nan
    p.data.copy_(new)
    p.grad = torch.zeros_like(p)
    opt.state[p]['exp_avg'].zero_()
    before = new.float()
    opt.step()
    got = p.detach().float()
    there = ~torch.isnan(before)                       # nothing else moves the weight: it rounds to what it was set to
    assert torch.equal(torch.isnan(got), ~there) and torch.equal(got[there], before[there])


def test_more_than_2_to_31_elements(dev):
    """offsets beyond 32 bits in parameters, gradients, codes and scales: the last elements against a tensor of their own"""
    from pde_surrogate_amd import optim
    n, tail = (1 << 31) + 2049, 4096 + 1              # (the tail begins at a block's start: the number before it is a multiple of 256)
    assert (n - tail) % 256 == 0
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device=dev))
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device=dev)
    q = torch.nn.Parameter(torch.randn(tail, device=dev).bfloat16())
    q.grad = torch.randn(tail, device=dev).bfloat16()
    p.data[-tail:], p.grad[-tail:] = q.data, q.grad
    norm = optim.clip_grad_norm_([p], math.inf)
    assert torch.equal(norm, optim.clip_grad_norm_([q], math.inf)) or abs(float(norm) / float(optim.clip_grad_norm_([q], math.inf)) - 1) < 4 * au.U
    a, b = optim.FusedAdamW([p], lr=1e-2, state_bits=8), optim.FusedAdamW([q], lr=1e-2, state_bits=8)
    a.step()
    b.step()
    assert torch.equal(p[-tail:], q) and not p[:-tail].any()
    sa, sb = a.state[p], b.state[q]
    assert torch.equal(sa['rms_scale'][-17:], sb['rms_scale']) and not sa['rms_scale'][:-17].any()
    # (the codes round by their own block numbers: equal to a spacing, not bit for bit)
    x, y = sa['rms_q'][-17 * 256:].float(), sb['rms_q'].float()
    assert ((x - y).abs() <= torch.maximum(y * 0.125, torch.full_like(y, 2.0 ** -9))).all()
    del a, sa
    c = optim.FusedAdamW([p], lr=1e-2)
    d = optim.FusedAdamW([q], lr=1e-2)
    c.step()
    d.step()
    assert torch.equal(p[-tail:], q) and torch.equal(c.state[p]['exp_avg_sq'][-tail:], d.state[q]['exp_avg_sq'])


# ---- lists, groups, states ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize('bits', [32, 8])
def test_gradients_that_come_and_go_and_many_groups(dev, bits):
    """every parameter counts its own steps; parameters without a gradient stay; more groups than one launch takes; mixed types"""
    from pde_surrogate_amd import optim
    ps = _params(dev, [300 + k for k in range(10)], 'float32') + _params(dev, [257] * 4, 'bfloat16')
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    a = optim.FusedAdamW([{'params': [p], 'lr': 1e-3 * (k + 1)} for k, p in enumerate(ps)], state_bits=bits)
    ones = [optim.FusedAdamW([q], lr=1e-3 * (k + 1), state_bits=bits) for k, q in enumerate(qs)]
    taken = [0] * len(ps)
    for t in range(5):
        _grads(ps, t)
        for k, (p, q) in enumerate(zip(ps, qs)):
            if (t + k) % 3 == 0 and t:
                p.grad = None
            else:
                q.grad = p.grad.clone()
                ones[k].step()
                taken[k] += 1
            if p.grad is None:
                q.grad = None
        a.step()
    for k, (p, q) in enumerate(zip(ps, qs)):
        assert float(a.state[p]['step']) == taken[k]
        if bits == 32:
            assert torch.equal(p, q)
        else:               # (another place in the list is another random sequence: rounding differs, the size of a step does not)
            assert float((p - q).detach().float().abs().max()) <= 5e-3 * (k + 1) * 5


@pytest.mark.parametrize('bits', [32, 8])
def test_a_thousand_tensors(dev, bits):
    """eleven launches and seven for the norm: all of them step by the one norm, as the same numbers do in one tensor"""
    from pde_surrogate_amd import optim
    flat = torch.randn(1000 * 256, device=dev)
    g = torch.randn_like(flat)
    ps = [torch.nn.Parameter(x.clone()) for x in flat.split(256)]
    one = torch.nn.Parameter(flat.clone())
    one.grad = g.clone()
    for p, x in zip(ps, g.split(256)):
        p.grad = x.clone()
    a, b = optim.FusedAdamW(ps, clip_norm=3.0, state_bits=bits), optim.FusedAdamW([one], clip_norm=3.0, state_bits=bits)
    for _ in range(2):
        a.step()
        b.step()
        assert torch.equal(a.grad_norm, b.grad_norm)
        if bits == 32 or _ == 0:               # (8-bit codes are rounded by the tensors' places)
            assert torch.equal(torch.cat([p.detach() for p in ps]), one.detach())
    n = optim.clip_grad_norm_(ps, 1.0)
    assert torch.equal(n, optim.clip_grad_norm_(one, 1.0)) and torch.equal(torch.cat([p.grad for p in ps]), one.grad)


def test_no_gradients_at_all_and_empty_tensors(dev):
    from pde_surrogate_amd import optim
    ps = _params(dev, [0, 0])
    opt = optim.FusedAdamW(ps, clip_norm=1.0)
    opt.step()
    assert float(opt.grad_norm) == 0.0
    for p in ps:
        p.grad = torch.zeros_like(p)
    opt.step()
    assert float(opt.grad_norm) == 0.0 and float(opt.state[ps[0]]['step']) == 1
    assert float(optim.clip_grad_norm_(ps, 1.0)) == 0.0


@pytest.mark.parametrize('bits,dtype,master', [(32, 'float32', False), (32, 'bfloat16', True), (8, 'float32', False), (8, 'bfloat16', True)])
def test_saved_and_copied_states_go_on_bit_for_bit(dev, tmp_path, bits, dtype, master):
    from pde_surrogate_amd import optim
    sizes = [5, 300, 1024, 4097]
    kw = dict(lr=1e-3, state_bits=bits, master_weights=master, seed=9, clip_norm=1.0)
    ps = _params(dev, sizes, dtype)
    a = optim.FusedAdamW(ps, **kw)
    for t in range(2):
        _grads(ps, t)
        a.step()
    torch.save(a.state_dict(), tmp_path / 'opt.pt')
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    b = optim.FusedAdamW(qs, **dict(kw, lr=9.0))
    b.load_state_dict(torch.load(tmp_path / 'opt.pt', map_location='cpu', weights_only=True))
    rs, c = copy.deepcopy((ps, a))
    assert b.param_groups[0]['lr'] == 1e-3 and c.state_bits == bits
    for t in range(2, 4):
        _grads(ps, t)
        for x in (qs, rs):
            for p, q in zip(ps, x):
                q.grad = p.grad.clone()
        for o in (a, b, c):
            o.step()
    for x, o in ((qs, b), (rs, c)):
        for p, q in zip(ps, x):
            assert torch.equal(p, q) and float(o.state[q]['step']) == 4
            for k in a.state[p]:
                assert torch.equal(a.state[p][k].reshape(-1).view(torch.uint8), o.state[q][k].reshape(-1).view(torch.uint8)), k


@pytest.mark.parametrize('ours', [False, True])
def test_states_of_an_optimiser_that_goes_the_other_way_are_refused(dev, ours):
    from pde_surrogate_amd import optim
    p, q = (torch.nn.Parameter(torch.ones(5, device=dev)) for _ in range(2))
    opt = optim.FusedAdamW([p], maximize=ours)
    with pytest.raises(ValueError, match='maximize'):
        opt.load_state_dict(torch.optim.AdamW([q], maximize=not ours).state_dict())
    opt.load_state_dict(torch.optim.AdamW([q], maximize=ours).state_dict())
    opt.load_state_dict(optim.FusedAdamW([q], maximize=ours).state_dict())
    p.grad = torch.ones_like(p)
    opt.step()
    assert ((p > 1) if ours else (p < 1)).all()


def test_saved_8_bit_states_load_into_their_own_memory_order_only(dev):
    from pde_surrogate_amd import optim
    x = torch.randn(8, 5, 3, 3, device=dev)
    a, b, c = (torch.nn.Parameter(y) for y in (x.to(memory_format=torch.channels_last), x.clone(), x.to(memory_format=torch.channels_last)))
    opts = [optim.FusedAdamW([p], state_bits=8) for p in (a, b, c)]
    for p, o in zip((a, b, c), opts):
        p.grad = torch.ones_like(p)
        o.step()
    sd = opts[0].state_dict()
    held, codes = b.detach().clone(), opts[1].state[b]['rms_q'].view(torch.uint8).clone()
    with pytest.raises(ValueError, match='memory order'):
        opts[1].load_state_dict(sd)
    assert torch.equal(opts[1].state[b]['rms_q'].view(torch.uint8), codes) and torch.equal(b, held)
    opts[2].load_state_dict(sd)
    for o, p in ((opts[0], a), (opts[2], c)):
        o.step()
    assert torch.equal(a, c) and 'order' not in opts[2].state[c]


def test_states_go_to_and_come_from_torch(dev):
    from pde_surrogate_amd import optim
    ps = _params(dev, [50, 3000])
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    a, b = optim.FusedAdamW(ps, lr=1e-3), torch.optim.AdamW(qs, lr=1e-3)
    for t in range(6):
        _grads(ps, t)
        for p, q in zip(ps, qs):
            q.grad = p.grad.clone()
        a.step()
        b.step()
        for p, q in zip(ps, qs):
            # each side rounds a handful of operations of an update of lr
            assert float((p - q).detach().abs().max()) <= 40 * au.U * (1e-3 * 10 + float(q.detach().abs().max()))
            assert float(a.state[p]['step']) == float(b.state[q]['step']) == t + 1
        if t == 1:
            saved = copy.deepcopy(b.state_dict())
            a = optim.FusedAdamW(ps, lr=1.0)
            a.load_state_dict(saved)
        if t == 3:
            saved = copy.deepcopy(a.state_dict())
            b = torch.optim.AdamW(qs, lr=1.0)
            b.load_state_dict(saved)
    before, keep = [p.detach().clone() for p in ps], a.state[ps[0]]['exp_avg'].clone()
    other = optim.FusedAdamW(ps, lr=1e-3, state_bits=8)
    for bad in (lambda: other.load_state_dict(a.state_dict()), lambda: a.load_state_dict(torch.optim.AdamW(qs, amsgrad=True).state_dict())):
        with pytest.raises(ValueError):
            bad()
    sd = a.state_dict()
    sd['state'][1]['exp_avg'] = sd['state'][1]['exp_avg'][:7]
    with pytest.raises(ValueError, match='shape'):
        a.load_state_dict(sd)
    assert torch.equal(a.state[ps[0]]['exp_avg'], keep) and torch.equal(ps[0], before[0])
    a.step()
    a.state = type(a.state)(dict)                     # a program that starts over
    a.step()
    assert float(a.state[ps[0]]['step']) == 1
    a.state.clear()
    a.step()
    assert float(a.state[ps[0]]['step']) == 1 and len(a.flat_state()['exp_avg']) == 1


# ---- streams, graphs ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('bits', [32, 8])
def test_two_optimisers_on_two_streams(dev, bits):
    from pde_surrogate_amd import optim
    sizes = [200_003] * 20
    want = []
    for seed in (1, 2):
        ps = _params(dev, sizes, seed=seed)
        _grads(ps, seed)
        opt = optim.FusedAdamW(ps, lr=1e-2, state_bits=bits, clip_norm=1.0)
        for _ in range(10):
            opt.step()
        want.append([p.detach().clone() for p in ps])
    torch.cuda.synchronize()
    both = []
    for seed in (1, 2):
        ps = _params(dev, sizes, seed=seed)
        _grads(ps, seed)
        both.append((ps, optim.FusedAdamW(ps, lr=1e-2, state_bits=bits, clip_norm=1.0), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(10):
        for ps, opt, s in both:
            with torch.cuda.stream(s):
                opt.step()
    torch.cuda.synchronize()
    for (ps, opt, s), w in zip(both, want):
        assert all(torch.equal(p, x) for p, x in zip(ps, w))


@pytest.mark.parametrize('bits,dtype,master', [(32, 'float32', False), (8, 'bfloat16', True)])
def test_captured_steps(dev, bits, dtype, master):
    """a captured step, replayed with new gradients and learning rates and eager work between the replays, is the eager one"""
    from pde_surrogate_amd import optim
    sizes = SIZES['many']
    kw = dict(state_bits=bits, master_weights=master, clip_norm=0.9, seed=3)
    ps, qs = _params(dev, sizes, dtype), _params(dev, sizes, dtype)
    lr = torch.tensor(1e-3, device=dev)
    a = optim.FusedAdamW([{'params': ps[:50]}, {'params': ps[50:], 'weight_decay': 0.0}], lr=lr, capturable=True, **kw)
    b = optim.FusedAdamW([{'params': qs[:50]}, {'params': qs[50:], 'weight_decay': 0.0}], lr=float(np.float32(1e-3)), **kw)
    for x in (ps, qs):
        _grads(x, 0)
    with pytest.raises(RuntimeError, match='eagerly'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            a.step()
    a.step()
    b.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    norm = a.grad_norm
    for t in range(1, 7):
        _grads(qs, t)
        for p, q in zip(ps, qs):
            p.grad.copy_(q.grad)
        lr.fill_(1e-3 / t)
        for g in b.param_groups:
            g['lr'] = float(np.float32(1e-3 / t))
        graph.replay()
        b.step()
        (torch.randn(1000, device=dev) * 2).sum().item()
        assert torch.equal(norm, b.grad_norm)
        for p, q in zip(ps, qs):
            assert torch.equal(p, q), t
            for k in a.state[p]:
                x, y = a.state[p][k], b.state[q][k]
                assert float(x) == float(y) == t + 1 if k == 'step' else torch.equal(x.reshape(-1).view(torch.uint8), y.reshape(-1).view(torch.uint8)), (t, k)
    with pytest.raises(RuntimeError, match='capturable'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            b.step()
    # an eager step of the same optimiser between replays, and clipping in a graph
    a.step()
    b.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    torch.cuda.synchronize()
    clip = torch.cuda.CUDAGraph()
    with torch.cuda.graph(clip):
        total = optim.clip_grad_norm_(ps, 0.5)
    for t in range(3):
        _grads(qs, 30 + t)
        for p, q in zip(ps, qs):
            p.grad.copy_(q.grad)
        clip.replay()
        want = optim.clip_grad_norm_(qs, 0.5)
        assert torch.equal(total, want) and all(torch.equal(p.grad, q.grad) for p, q in zip(ps, qs))


@pytest.mark.parametrize('bits', [32, 8])
def test_an_infinite_limit_changes_nothing(dev, bits):
    """clip_norm = inf finds the norm of every step; a norm that is infinite or NaN leaves the other elements alone"""
    from pde_surrogate_amd import optim
    ps, qs = _params(dev, [300, 40]), _params(dev, [300, 40])
    a, b = optim.FusedAdamW(ps, clip_norm=math.inf, state_bits=bits), optim.FusedAdamW(qs, state_bits=bits)
    for x in (1.0, math.inf, math.nan):
        _grads(ps, 1)
        ps[0].grad[5] = x
        for p, q in zip(ps, qs):
            q.grad = p.grad.clone()
        a.step()
        b.step()
        norm = float(a.grad_norm)
        assert math.isnan(norm) if math.isnan(x) else norm == math.inf if math.isinf(x) else norm > 1
        for p, q in zip(ps, qs):
            assert torch.equal(p.isnan(), q.isnan()) and torch.equal(p[~p.isnan()], q[~q.isnan()])
    a.clip_norm = None
    a.step()
    assert a.grad_norm is None


def test_autograd_sees_the_step(dev):
    """a parameter changed between a forward and its backward is caught, as with any in-place change"""
    from pde_surrogate_amd import optim
    p = torch.nn.Parameter(torch.randn(5, device=dev))
    opt = optim.FusedAdamW([p])
    y = (p * p).sum()
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward()
    assert opt.step(lambda: 3.5) == 3.5


def test_closures_schedulers_and_tied_parameters(dev):
    from pde_surrogate_amd import optim
    w = torch.nn.Parameter(torch.randn(20, 20, device=dev) * 0.1)
    opt = optim.FusedAdamW([w], lr=1.0)
    sched = torch.optim.lr_scheduler.OneCycleLR(opt, max_lr=1e-2, total_steps=10)

    def closure():
        opt.zero_grad()
        loss = ((w @ w) ** 2).sum() + w.sum()          # used twice: gradients add up
        loss.backward()
        return loss
    first = float(opt.step(closure))
    for _ in range(5):
        sched.step()
        last = float(opt.step(closure))
    assert math.isfinite(first) and math.isfinite(last) and torch.isfinite(w).all()
    flat = torch.zeros(10, device=dev)
    two = [torch.nn.Parameter(flat[:5]), torch.nn.Parameter(flat[:5])]
    for p in two:
        p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError, match='share their memory'):
        optim.FusedAdamW(two).step()
    with pytest.raises(ValueError, match='share their memory'):
        optim.clip_grad_norm_([two[0], two[0]], 1.0)
    two = [torch.nn.Parameter(flat[:6]), torch.nn.Parameter(flat[5:])]             # one element in common
    g = torch.zeros(11, device=dev)
    two[0].grad, two[1].grad = g[:6], g[5:10]
    with pytest.raises(RuntimeError, match='share their memory'):
        optim.FusedAdamW(two).step()
    with pytest.raises(ValueError, match='share their memory'):
        optim.clip_grad_norm_(two, 1.0)
    two[1].grad = g[6:]
    optim.clip_grad_norm_(two, 1.0)


def test_refusals(dev):
    from pde_surrogate_amd import optim
    p = torch.nn.Parameter(torch.zeros(4, 4, device=dev))
    with pytest.raises(RuntimeError, match='float32, bfloat16 or float16'):
        optim.FusedAdamW([torch.nn.Parameter(torch.zeros(3, dtype=torch.float64, device=dev))])
    with pytest.raises(ValueError, match='not dense'):
        optim.FusedAdamW([torch.nn.Parameter(torch.zeros(4, 8, device=dev)[:, ::2])])
    with pytest.raises(ValueError, match='tensor'):
        optim.FusedAdamW([p], lr=torch.tensor(1e-3))
    with pytest.raises(ValueError, match='float16'):
        optim.FusedAdamW([torch.nn.Parameter(torch.zeros(3, dtype=torch.float16, device=dev))], master_weights=True)
    for lr in (torch.tensor(1e-3), torch.tensor([1e-3], device=dev), torch.tensor(1e-3, device=dev, dtype=torch.float64)):
        with pytest.raises(ValueError, match='0-d float32'):
            optim.FusedAdamW([p], lr=lr, capturable=True)
    opt = optim.FusedAdamW([p], lr=1e-3, capturable=True)
    opt.param_groups[0]['lr'] = torch.tensor(1e-3)                                  # a host tensor put there later
    p.grad = torch.ones_like(p)
    with pytest.raises(ValueError, match='0-d float32'):
        opt.step()
    assert not p.any()
    optim.FusedAdamW([{'params': []}]).step()
    opt = optim.FusedAdamW([p])
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        opt.add_param_group({'params': [torch.nn.Parameter(torch.zeros(3))]})
    assert len(opt.param_groups) == 1
    p.grad = torch.ones_like(p)
    opt.step()
    keep = p.detach().clone()
    p.grad = None
    p.data = torch.zeros(5, 5, device=dev)
    p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError, match='another size'):
        opt.step()
    p.grad = None
    p.data = torch.zeros(4, 4)
    p.grad = torch.ones(4, 4)
    with pytest.raises(RuntimeError, match='no longer'):
        opt.step()
    p.grad = None
    p.data = keep.half()
    p.grad = torch.ones(4, 4, device=dev, dtype=torch.float16)
    with pytest.raises(RuntimeError, match='no longer'):
        opt.step()
    p.grad = None
    p.data = keep
    p.grad = torch.ones(4, 4, device=dev).to_sparse()
    with pytest.raises(RuntimeError, match='sparse'):
        opt.step()
    with pytest.raises(RuntimeError, match='sparse'):
        optim.clip_grad_norm_([p], 1.0)
    with pytest.raises(ValueError, match='norm_type'):
        optim.clip_grad_norm_([p], 1.0, 1.0)
    with pytest.raises(ValueError, match='negative'):
        optim.clip_grad_norm_([p], -1.0)


@pytest.mark.parametrize('optimizer,clip', [('adam', '0.5'), ('adamw', None), ('adamw', '0.5'), ('adamw8', '0.5')])
def test_cli_runs(dev, tmp_path, monkeypatch, optimizer, clip):
    """the training script with each optimiser: it runs, writes its files and the loss is finite"""
    import json
    import train_codec_mixed_residual as t
    from pde_surrogate_amd import optim
    monkeypatch.setenv('WORLD_SIZE', '1')
    calls = []
    for name, cls in (('Adam', optim.Adam), ('FusedAdamW', optim.FusedAdamW)):
        real = cls.step
        monkeypatch.setattr(cls, 'step', lambda self, *a, _r=real, _n=name, **k: (calls.append(_n), _r(self, *a, **k))[1])
    argv = ['--exp-dir', str(tmp_path), '--ntrain', '32', '--ntest', '16', '--batch-size', '8', '--test-batch-size', '8', '--epochs', '2',
            '--ckpt-freq', '2', '--cuda', '0', '--synthetic', '--blocks', '111', '--growth-rate', '8', '--init-features', '16',
            '--weight-decay', '0.01', '--mode', 'dropin', '--optimizer', optimizer] + (['--clip-norm', clip] if clip else [])
    with contextlib.redirect_stdout(io.StringIO()):
        t.main(argv)
    run = tmp_path / 'codec/mixed_residual/grf_kle512_ntrain32_run1_bs8_lr0.001_epochs2'
    lt = np.loadtxt(run / 'training/loss_train.txt')
    assert lt.shape == (2,) and np.isfinite(lt).all()
    assert json.load(open(run / 'args.txt'))['optimizer'] == optimizer
    assert calls == ['Adam' if optimizer == 'adam' else 'FusedAdamW'] * 8


def test_the_flat_adam_of_a_network_goes_on_after_clipping(dev, monkeypatch):
    """clip_grad_norm_ works in place on the views that the network's backward returned: optim.Adam still takes its one-launch step,
    and equals torch.optim.Adam fed the clipped gradients"""
    from pde_surrogate_amd import _lib, optim
    from pde_surrogate_amd.models.codec import DenseED
    torch.manual_seed(2)
    with contextlib.redirect_stdout(io.StringIO()):
        net = DenseED(1, 3, 32, [1, 1, 1], growth_rate=8, init_features=16).to(dev)
    opt = optim.Adam(net.parameters(), lr=1e-3)
    L, count = _lib.lib(), []
    real = L.pdes_adam_step_host

    class Spy:
        def __getattr__(self, k):
            if k == 'pdes_adam_step_host':
                count.append(1)
                return real
            return getattr(L, k)
    monkeypatch.setattr(_lib, '_lib', Spy())
    for t in range(3):
        net.zero_grad()
        net(torch.rand(4, 1, 32, 32, device=dev)).square().mean().backward()
        before = [p.grad.clone() for p in net.parameters()]
        norm = optim.clip_grad_norm_(net.parameters(), 1e-3)
        want = math.sqrt(sum(float((au.f64(g) ** 2).sum()) for g in before))
        assert want > 1e-3 and abs(float(norm) / want - 1) <= 1.001 * au.U
        for p, g in zip(net.parameters(), before):
            au.within(p.grad, au.f64(g) * 1e-3 / (want + 1e-6), np.abs(au.f64(g)) * 1e-3 / want * 6 * au.U + au.TINY, 'clipped')
        opt.step()
    assert len(count) == 3
