"""CPU tests of the list optimiser and of clipping: refusals (arguments, the C entries' own checks, which return before any
launch), the memory-order helpers, and the random numbers of the 8-bit states' rounding."""
import ctypes
import math

import numpy as np
import pytest
import torch

import adamw_util as au


@pytest.fixture(scope='module', autouse=True)
def _built():
    from pde_surrogate_amd import build
    build.build(verbose=False)                 # (nothing to do where everything is built)


def test_arguments_are_checked_before_anything_else():
    from pde_surrogate_amd import optim
    p = [torch.nn.Parameter(torch.zeros(3))]
    for kw in (dict(state_bits=16), dict(clip_norm=-1.0), dict(clip_norm=math.nan), dict(seed=-1), dict(seed=1 << 32)):
        with pytest.raises(ValueError):
            optim.FusedAdamW(p, **kw)
    for kw in (dict(lr=-1.0), dict(lr=math.nan), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0), dict(weight_decay=-0.1),
               dict(lr=torch.tensor(0.1))):
        with pytest.raises(ValueError):
            optim.FusedAdamW(p, **kw)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        optim.FusedAdamW(p)
    with pytest.raises(RuntimeError, match='float32, bfloat16 or float16'):
        optim.FusedAdamW([torch.nn.Parameter(torch.zeros(3, dtype=torch.float64))])
    p[0].grad = torch.ones(3)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        optim.clip_grad_norm_(p, 1.0)
    with pytest.raises(ValueError, match='norm_type'):
        optim.clip_grad_norm_(p, 1.0, 3.0)
    for bad in (-0.5, math.nan):
        with pytest.raises(ValueError, match='negative'):
            optim.clip_grad_norm_(p, bad)
    p[0].grad = None
    assert float(optim.clip_grad_norm_(p, 1.0)) == 0.0


def test_torch_optimisers_are_still_the_modules_own():
    from pde_surrogate_amd import optim
    assert optim.AdamW is torch.optim.AdamW and optim.SGD is torch.optim.SGD and issubclass(optim.Adam, torch.optim.Adam)
    assert issubclass(optim.FusedAdamW, torch.optim.Optimizer)


def test_memory_order_helpers():
    from pde_surrogate_amd.adamw import _dense, _order, _overlap, _same_order
    x = torch.zeros(4, 6, 2)
    assert _dense(x) and _dense(x.permute(2, 0, 1)) and _dense(x[1]) and _dense(torch.zeros(())) and _dense(torch.zeros(0, 3))
    assert not _dense(x[:, ::2]) and not _dense(x[:, :3]) and not _dense(torch.zeros(1, 1).expand(3, 3)) and not _dense(x.as_strided((3, 3), (1, 1)))
    assert _same_order(x, torch.ones(4, 6, 2)) and not _same_order(x, torch.ones(6, 4, 2).permute(1, 0, 2))
    assert _same_order(torch.zeros(1, 5), torch.zeros(5, 1).t())
    assert _order(x) == (0, 1, 2) and _order(x.permute(2, 0, 1)) == (1, 2, 0) and _order(torch.zeros(())) == ()
    assert _order(torch.zeros(1, 5)) == _order(torch.zeros(5, 1).t()) == (1,)
    assert _overlap([(8, 4), (8, 8)]) and _overlap([(20, 8), (8, 13)]) and not _overlap([(20, 8), (8, 12), (0, 0), (0, 0), (10, 0)])


def test_c_entries_refuse_what_the_kernels_do_not_take():
    """every call here is rejected on the host: none reaches a launch"""
    from pde_surrogate_amd import _lib
    from pde_surrogate_amd.adamw import AdamWClass, AdamWState, MtTensor
    L = _lib.lib()
    EINVAL, EALIGN = -1, -3
    one = (ctypes.c_ulonglong * 1)(4096)
    n = (ctypes.c_longlong * 1)(10)
    norm = L.pdes_grad_norm
    assert norm(one, n, 1, 0, 2, None, 0, None) == EINVAL
    assert norm(one, n, 1, 3, 2, 4096, 0, None) == EINVAL
    assert norm(one, n, 1, 0, 1, 4096, 0, None) == EINVAL
    assert norm(None, n, 1, 0, 2, 4096, 0, None) == EINVAL
    assert norm(one, n, -1, 0, 2, 4096, 0, None) == EINVAL
    assert norm((ctypes.c_ulonglong * 1)(4098), n, 1, 0, 2, 4096, 0, None) == EALIGN
    assert norm((ctypes.c_ulonglong * 1)(4097), n, 1, 1, 2, 4096, 0, None) == EALIGN
    assert norm((ctypes.c_ulonglong * 1)(0), n, 1, 0, 2, 4096, 0, None) == EINVAL
    for bad in (-1, 1 << 40):
        assert norm(one, (ctypes.c_longlong * 1)(bad), 1, 0, 2, 4096, 0, None) == EINVAL
    for limit in (-1.0, math.nan):
        assert L.pdes_clip_grads(one, n, 1, 0, 2, 4096, limit, None, None) == EINVAL
    assert L.pdes_clip_grads(one, n, 1, 0, 2, None, 1.0, None, None) == EINVAL

    def step(params=4096, grads=4096, count=1, nclasses=1, tensor=(10, 0, 0, 0), cls=(1e-3, 0.9, 0.99, 1e-8, 0.0, 1, None, None), **state):
        st = AdamWState(exp_avg=4096, exp_avg_sq=4096, exp_avg_scale=4096, rms_scale=4096, blocks=1, dtype=0, bits=32)
        for k, v in state.items():
            setattr(st, k, v)
        return L.pdes_adamw_step((ctypes.c_ulonglong * 1)(params), (ctypes.c_ulonglong * 1)(grads), (MtTensor * 1)(MtTensor(*tensor)), count,
                                 (AdamWClass * 1)(AdamWClass(*cls)), nclasses, ctypes.byref(st), None)
    for kw in (dict(count=-1), dict(nclasses=0), dict(nclasses=9), dict(bits=16), dict(dtype=3), dict(low=4096), dict(blocks=0), dict(blocks=-1),
               dict(params=0), dict(grads=0), dict(exp_avg=None), dict(exp_avg_sq=None), dict(bits=8, rms_scale=None),
               dict(tensor=(257, 0, 0, 0)), dict(tensor=(10, 1, 0, 0)), dict(tensor=(10, -1, 0, 0)), dict(tensor=(10, (1 << 63) - 1, 0, 0)), dict(tensor=(-1, 0, 0, 0)),
               dict(tensor=(10, 0, 1, 0)), dict(tensor=(10, 0, -1, 0)), dict(norm_rows=4096, limit=-1.0), dict(norm_rows=4096, limit=math.nan),
               dict(cls=(1e-3, 1.0, 0.99, 1e-8, 0.0, 1, None, None)), dict(cls=(1e-3, 0.9, math.nan, 1e-8, 0.0, 1, None, None)),
               dict(cls=(1e-3, 0.9, 0.99, -1.0, 0.0, 1, None, None)), dict(cls=(1e-3, 0.9, 0.99, 1e-8, 0.0, 0, None, None)),
               dict(cls=(1e-3, 0.9, 0.99, 1e-8, 0.0, 1, 4096, None)), dict(cls=(1e-3, 0.9, 0.99, 1e-8, 0.0, 1, None, 4096))):
        assert step(**kw) == EINVAL, kw
    for kw in (dict(params=4098), dict(grads=4097), dict(exp_avg=4100), dict(exp_avg_sq=4104), dict(dtype=1, low=4098), dict(dtype=1, params=4097)):
        assert step(**kw) == EALIGN, kw


def test_mirrors_have_the_size_of_the_c_structures():
    from pde_surrogate_amd import _lib, adamw
    for which, cls in ((9, adamw.MtTensor), (10, adamw.AdamWClass), (11, adamw.AdamWState)):
        assert _lib.lib().pdes_sizeof(which) == ctypes.sizeof(cls)


def test_the_rounding_numbers_are_even_and_unrelated():
    """400,000 numbers of each kind: mean, every bit's share (5 standard errors: 0.5 / sqrt(N) = 8e-4), and correlations (5 / sqrt(N)
    = 8e-3) between an element's two numbers, neighbours, steps, tensors and seeds"""
    a, b = au.dither(7, 100, 3, 1600)
    n = a.size
    for x in (a, b):
        assert x.min() >= 0 and x.max() < 1 << 20
        assert abs(x.mean() / (1 << 20) - 0.5) < 5 * 0.2887 / math.sqrt(n)
        for bit in range(20):
            assert abs(((x >> bit) & 1).mean() - 0.5) < 5 * 0.5 / math.sqrt(n), bit
        counts = np.bincount((x >> 12).reshape(-1), minlength=256)
        assert ((counts - n / 256) ** 2).sum() / (n / 256) < 255 + 5 * math.sqrt(2 * 255)      # chi squared of the upper byte

    def corr(x, y):
        return abs(np.corrcoef(x.reshape(-1), y.reshape(-1))[0, 1])
    lim = 5 / math.sqrt(n)
    assert corr(a, b) < lim
    assert corr(a[:, 1:], a[:, :-1]) < lim * 1.01 and corr(b[1:], b[:-1]) < lim * 1.01
    for other in (au.dither(7, 101, 3, 1600), au.dither(7, 100, 4, 1600), au.dither(8, 100, 3, 1600)):
        assert corr(a, other[0]) < lim and corr(b, other[1]) < lim


def test_held_values_are_within_a_spacing_and_right_on_average():
    """the definition itself: e4m3's spacing is 2^-3 of the binade (2^-9 under 2^-6), rounding goes to one of the two neighbours, and
    on average to the value (0.2 % of it over 2000 draws: the standard error of a spacing of 12.5 % is 0.14 %, three of them)"""
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((64, 256)) * np.exp(rng.standard_normal((64, 256)) * 3)).astype(np.float32)
    total = np.zeros(x.shape)
    times = 2000
    for t in range(times):
        noise, _ = au.dither(1, t, 0, 64)
        code, scale = au.held(x, noise, False)
        value = torch.from_numpy(code.copy()).view(torch.float8_e4m3fn).float().numpy() * scale[:, None]
        if t < 5:
            y = np.abs(x) / scale[:, None].astype(np.float64)
            spacing = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(y, 1e-30))), -6) - 3)
            assert (np.abs(value - x) <= spacing * scale[:, None] * (1 + 1e-6)).all()
            assert (np.sign(value) * np.sign(x) >= 0).all()
        total += value
    top = np.abs(x).max(1, keepdims=True)
    big = np.abs(x) > top * 2.0 ** -12                     # (smaller ones are held by chance alone)
    rel = (total / times - x)[big] / np.abs(x)[big]
    assert abs(rel.mean()) < 5e-4 and (np.abs(rel) < 5 * 0.0625 / math.sqrt(times) * np.maximum(1, 2.0 ** -6 * top.repeat(256, 1)[big] / 448 * 448 / np.abs(x)[big] * 8)).mean() > 0.99


def test_cli_flags(tmp_path):
    """--optimizer and --clip-norm belong to --mode dropin; refused before a directory is made"""
    import train_codec_max_likelihood as m
    import train_codec_mixed_residual as t
    for cli in (t, m):
        a = cli.Parser().parse(['--exp-dir', str(tmp_path / 'ok'), '--mode', 'dropin', '--optimizer', 'adamw8', '--clip-norm', '0.5'])
        assert (a.optimizer, a.clip_norm) == ('adamw8', 0.5)
        a = cli.Parser().parse(['--exp-dir', str(tmp_path / 'ok')])
        assert (a.optimizer, a.clip_norm) == ('adam', None)
        for argv in (['--optimizer', 'adamw'], ['--clip-norm', '1'], ['--mode', 'dropin', '--clip-norm', '-1'],
                     ['--mode', 'dropin', '--clip-norm', 'nan'], ['--mode', 'dropin', '--optimizer', 'sgd']):
            with pytest.raises(SystemExit):
                cli.Parser().parse(['--exp-dir', str(tmp_path / 'no')] + argv)
    assert not (tmp_path / 'no').exists()


def test_host_functions_on_lists():
    """_tensor_list.so on CPU tensors: patterns of gradients, version counters, and no address of anything that is not on the device"""
    from pde_surrogate_amd.adamw import _host, _words
    host = _host()
    ps = [torch.nn.Parameter(torch.zeros(3)) for _ in range(4)]
    ps[1].grad, ps[3].grad = torch.ones(3), torch.ones(3)
    mask = bytes([0, 1, 0, 1])
    assert host.fits([ps], ps, mask) and host.fits([ps[:1], [], ps[1:]], ps, mask)
    assert not host.fits([ps[:3]], ps, mask) and not host.fits([ps + ps[:1]], ps, mask) and not host.fits([ps[::-1]], ps, mask)
    assert not host.fits([ps], ps, bytes([0, 1, 1, 1])) and not host.fits([ps], ps, bytes(4))
    before = [p._version for p in ps] + [ps[1].grad._version]
    host.changed(ps, False)
    assert [p._version for p in ps] == [v + 1 for v in before[:4]] and ps[1].grad._version == before[4]
    host.changed(ps, True)
    assert ps[1].grad._version == before[4] + 1 and [p._version for p in ps] == [v + 1 for v in before[:4]]
    (sizes, at), (out, oat), (gout, gat) = _words(4), _words(4), _words(4)
    assert host.gather(ps, ps, 0, 0, at, oat, gat) == 0 and not any(out)
    assert host.gather([], [], 0, 0, at, oat, gat) == -1
    (a, aat), (b, bat) = _words(12), _words(12)
    assert host.gradients(ps, aat, bat)[4] == 1 and host.gradients([ps[0]], aat, bat) == (0, 0, 0, -1, -1, 0)
    for bad in (lambda: host.gather((), ps, 0, 0, at, oat, gat), lambda: host.gather(ps, [], 0, 0, at, oat, gat), lambda: host.gather(ps),
                lambda: host.gradients(None, aat, bat), lambda: host.fits([ps], ps, b''), lambda: host.fits(ps, ps, mask), lambda: host.changed(3, 1)):
        with pytest.raises(TypeError):
            bad()
