"""Plain computations that the AdamW / clipping tests compare with: one step in 64 bits from given inputs together with how
far fp32 arithmetic may be off, and the 8-bit states' codes from the definition in numpy."""
import math

import numpy as np

BLOCK = 256
U = 2.0 ** -24                                  # half a step of fp32, relative
HALF = {'float32': 0.0, 'bfloat16': 2.0 ** -8, 'float16': 2.0 ** -11}
TINY = 2.0 ** -148


def f64(t):
    return t.detach().cpu().double().numpy().reshape(-1)


def step64(w, g, m, v, t, lr, betas, eps, wd, factor=1.0):
    """(w, m, v) in 64 bits from 64-bit inputs, and the bounds (w, m, v) of a computation in fp32 that rounds the
    constants and each operation once.  With u = 2^-24:
      m: constant, product, sum: 3 u of each term's size            -> 4 u M, M = |b1 m| + |(1 - b1) g|
      v: constant, square, product, sum: 4 u                          -> 5 u v
      denominator: sqrt halves 5 u and adds u, constant, product, eps and sum add 4 u -> 8 u of it
      quotient and step: (4 u M + 9 u |m|) / den, and 2 u more        -> 15 u s M / den
      weight: constant, product, difference 3 u |w|, and u of the change
    a clipping factor off by 4 u (norm, sum, reciprocal, product) and its product move g by 5 u, so m by 5 u and v by 10 u"""
    b1, b2 = betas
    extra = 0 if factor == 1.0 else 5
    g = g * factor
    big = np.abs(b1 * m) + np.abs((1 - b1) * g)
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    den = np.sqrt(v) / math.sqrt(1 - b2 ** t) + eps
    s = lr / (1 - b1 ** t)
    with np.errstate(all='ignore'):
        change = s * np.where(m == 0, 0.0, m / den)
        size = s * np.where(big == 0, 0.0, big / den)
    new = w * (1 - lr * wd) - change
    return (new, m, v), (4 * U * np.abs(w) + (17 + 2 * extra) * U * size + TINY, (4 + extra) * U * big + TINY, (5 + 2 * extra) * U * v + TINY)


def within(got, want, bound, what):
    got = f64(got) if not isinstance(got, np.ndarray) else got
    assert got.shape == want.shape, what
    off = np.abs(got - want) - bound
    assert np.all(off <= 0), f'{what}: {int((off > 0).sum())} of {off.size} beyond the bound, worst {np.nanmax(off)} at {int(np.nanargmax(off))}'


def master64(p, low):
    """bf16 parameters and the 16 bits below them -> the fp32 weights, as 64-bit"""
    import torch
    bits = (p.detach().cpu().reshape(-1).view(torch.int16).to(torch.int32) << 16) + low.detach().cpu().reshape(-1).to(torch.int32)
    return bits.view(torch.float32).double().numpy()


def mix(x):
    x = np.asarray(x, np.uint64) & np.uint64(0xffffffff)
    m = np.uint64(0xffffffff)
    x = x ^ (x >> np.uint64(16))
    x = (x * np.uint64(0x6A09E667)) & m
    x = x ^ (x >> np.uint64(15))
    x = (x * np.uint64(0xBB67AE85)) & m
    return x ^ (x >> np.uint64(16))


def dither(seed, t, ordinal, blocks):
    """the two 20-bit numbers of every element of a tensor's blocks"""
    gold = np.uint64(0x9E3779B9)
    key = mix(np.uint64(seed) + gold * np.uint64(t))
    key = mix(key + gold * np.uint64(ordinal + 1))
    key = mix(key + gold * np.arange(blocks, dtype=np.uint64))
    h = mix(key[:, None] + gold * np.arange(BLOCK, dtype=np.uint64)[None])
    return (h >> np.uint64(12)).astype(np.int64), (h & np.uint64(0xfffff)).astype(np.int64)


def held(x, noise, root):
    """(codes as uint8, scales) of fp32 rows x [blocks, 256], non-finite values included, from the definition in fp32: x times 448 /
    largest, cut to multiples of 2^-29 under 2^-6 (2^-20 of a spacing there), plus the noise, rounded down"""
    mag = np.abs(x)
    fine = np.isfinite(x)
    top = np.where(fine, mag, np.float32(0)).max(1, keepdims=True)
    live = top >= np.float32(2.0 ** -100)
    with np.errstate(all='ignore'):
        inverse = np.where(live, np.float32(448) / top, np.float32(0)).astype(np.float32)
        y = np.minimum((np.where(fine, mag, np.float32(0)) * inverse).astype(np.float32), np.float32(448))
        y = np.where(y < 2.0 ** -6, np.floor(y * np.float32(2.0 ** 29)) * np.float32(2.0 ** -29), y).astype(np.float32)
        y = (y * np.float32(2.0 ** -120)).astype(np.float32)
    code = np.minimum((y.view(np.int32).astype(np.int64) + noise) >> 20, 0x7e)
    if root:
        code = np.where((code == 0) & (x > 0), 1, code)
    code = np.where(fine, code, 0x7f)
    if not root:
        code = code | np.where(np.signbit(x), 0x80, 0)
    return code.astype(np.uint8), np.where(live, top * np.float32(1 / 448), np.float32(0)).astype(np.float32)[:, 0]


def rows(x, n):
    """fp32 [blocks, 256] of n values, zeros behind them"""
    blocks = -(-n // BLOCK)
    out = np.zeros(blocks * BLOCK, np.float32)
    out[:n] = np.asarray(x, np.float32).reshape(-1)
    return out.reshape(blocks, BLOCK)


def step8(w, g, mq, ms, rq, rs, t, lr, betas, eps, wd, seed, ordinal, factor=np.float32(1)):
    """one step with 8-bit states in fp32, one rounding per operation: (w, the size of the terms that
    its change by the gradient is made of, m codes, m scales, r codes, r scales).  mq / rq: the held values [blocks, 256] as fp32; w, g fp32 [n]"""
    f = np.float32
    b1, b2 = betas
    n = w.size
    with np.errstate(all='ignore'):
        gr = rows(g, n) * f(factor)
        m = mq * ms[:, None] * f(b1) + gr * f(1 - b1)
        r = rq * rs[:, None]
        r = np.sqrt(r * r * f(b2) + gr * gr * f(1 - b2))
        for_m, for_r = dither(seed, t, ordinal, m.shape[0])
        out = held(m, for_m, False) + held(r, for_r, True)
        u = m / (r * f(1 / math.sqrt(1 - b2 ** t)) + f(eps))
        step = f(lr / (1 - b1 ** t))
        new = rows(w, n) * f(1 - lr * wd) - u * step
        size = (np.abs(mq * ms[:, None]) * b1 + np.abs(gr) * (1 - b1)) / (r * (1 / math.sqrt(1 - b2 ** t)) + eps) * step
    assert new.dtype == np.float32
    return (new.reshape(-1)[:n], size.reshape(-1)[:n]) + out


def value(codes):
    """what e4m3 codes stand for"""
    import torch
    return torch.from_numpy(np.ascontiguousarray(codes)).view(torch.float8_e4m3fn).double().numpy()


def codes_near(got, want, what):
    """Codes of roots that are the neighbouring fp32 number in one case of two million: such a one takes the neighbouring code with a
    chance of 2^-23 / 2^-4.  So one code of a tensor may differ, or 2^-20 of them, by one spacing (2^-3 of the larger value, or 2^-9)."""
    x, y = value(got), value(want)
    assert np.all(np.abs(x - y) <= np.maximum(np.maximum(np.abs(x), np.abs(y)) / 8, 2.0 ** -9)), what
    assert np.count_nonzero(x != y) <= max(1, x.size * 2.0 ** -20), f'{what}: {np.count_nonzero(x != y)} of {x.size} codes differ'
