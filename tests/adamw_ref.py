"""CPU restatement of gs_adamw_step, gs_grad_norm and the 8-bit moment format
(include/gsb200.h): moments in explicit float32 roundings, codes from their
definition in values (float64), parameters in float64."""
import math

import numpy as np

BLOCK = 128
GOLDEN = 0x9E3779B9
F32 = np.float32


def mix32(x):
    x = np.asarray(x, dtype=np.uint64) & 0xFFFFFFFF
    x = x ^ (x >> np.uint64(16))
    x = (x * np.uint64(0x7FEB352D)) & np.uint64(0xFFFFFFFF)
    x = x ^ (x >> np.uint64(15))
    x = (x * np.uint64(0x846CA68B)) & np.uint64(0xFFFFFFFF)
    return x ^ (x >> np.uint64(16))


def noise(seed, count, tensor, n, start=0):
    """The 32-bit hashes of elements [start, start + n) of a tensor."""
    key = mix32((seed + GOLDEN * count) & 0xFFFFFFFF)
    key = mix32((int(key) + GOLDEN * tensor) & 0xFFFFFFFF)
    e = np.arange(start, start + n, dtype=np.uint64)
    bkey = mix32(np.uint64(int(key)) ^ (e // BLOCK))
    return mix32((bkey + np.uint64(GOLDEN) * (e % BLOCK)) & np.uint64(0xFFFFFFFF))


def _top(signed):
    return (15, 127) if signed else (31, 255)


def decode(codes, exps, signed):
    """Float64 values of codes."""
    c = codes.astype(np.int64)
    mag = c % 128 if signed else c
    ex, frac = mag // 8, (mag % 8) / 8.0
    val = np.where(ex == 0, np.ldexp(frac, 1 - _top(signed)[0]), np.ldexp(1.0 + frac, ex - _top(signed)[0]))
    f = np.repeat(exps.astype(np.int64), BLOCK)[:c.size]
    val = np.ldexp(val, f - 127)
    val = np.where(f == 255, np.nan, val)
    return np.where(c > 127, -val, val) if signed else val


def block_exponents(x):
    """The exponent bytes of float32 values (padded with zeros to whole blocks)."""
    pad = -x.size % BLOCK
    bits = np.abs(np.concatenate([x, np.zeros(pad, F32)])).view(np.uint32).reshape(-1, BLOCK).max(1)
    return np.minimum((bits.astype(np.uint64) + 0xFFFFF) >> np.uint64(23), 255).astype(np.uint8)


def encode(x, u, signed):
    """(codes, exponent bytes) of float32 values: magnitudes are multiples of a
    step that depends on their octave, the multiple below, or the one above
    when the remainder plus u (in [0, 1)) reaches a whole step."""
    exps = block_exponents(x)
    f = np.repeat(exps.astype(np.int64), BLOCK)[:x.size]
    bottom, most = 1 - _top(signed)[0], _top(signed)[1]
    with np.errstate(all="ignore"):
        a = np.where(f == 255, 0.0, np.ldexp(np.abs(x.astype(np.float64)), 127 - f))
    octave = np.maximum(np.frexp(np.maximum(a, 1e-300))[1] - 1, bottom)
    # magnitudes below 2^-126 of float32 after scaling keep 23 digits there: 2^-20 of a step
    a = np.where(octave == bottom, np.round(np.ldexp(a, 23 - bottom)) / 2.0 ** (23 - bottom), a)
    k = np.floor(np.ldexp(a, 3 - octave) + u).astype(np.int64)  # in eighths of the octave
    over = k >= 16
    octave, k = octave + over, np.where(over, k // 2, k)
    code = np.minimum(np.where(k >= 8, (octave - bottom) * 8 + k, k), most)
    if signed:
        code = code | (np.signbit(x).astype(np.int64) << 7)
    else:
        code = np.where((x > 0) & (code == 0), 1, code)
    return np.where(f == 255, 0, code).astype(np.uint8), exps


def moments(m, v, g, scale, b1, b2):
    """(m', v') in float32, each product and sum rounded."""
    with np.errstate(all="ignore"):
        g = (g.astype(F32) * F32(scale)).astype(F32)
        m = (m.astype(F32) * F32(b1)).astype(F32) + (g * F32(1.0 - b1)).astype(F32)
        v = (v.astype(F32) * F32(b2)).astype(F32) + ((g * g).astype(F32) * F32(1.0 - b2)).astype(F32)
    return m.astype(F32), v.astype(F32)


def param(p, m, v, count, lr, wd, b1, b2, eps, active=None):
    """p' in float64 and a bound of the float32 kernel's error.

    Relative roundings u = 2^-24 of the update's factors, counted upwards:
    1 - b1^t and 1 - b2^t by expm1 (argument 2, function 4, reciprocal 1: 7
    each, the second under a square root), the product with each (1), the
    approximate square root (4), + eps (1), the approximate quotient (4), lr
    (exponent's argument up to 5 x 2 x 2, function 4: 24), two products and one
    sum (3): at most 56 u of the update; the weight decay's part takes part in the
    last ones (30 u); p itself one rounding of the result (1 u, taken as 2)."""
    u = 2.0 ** -24
    with np.errstate(all="ignore"):
        m, v, p = m.astype(np.float64), v.astype(np.float64), p.astype(np.float64)
        t = count + 1
        upd = m / (1.0 - b1 ** t) / (np.sqrt(v / (1.0 - b2 ** t)) + eps)
        new = p - lr * (upd + wd * p)
        err = 2 * u * np.abs(new) + abs(lr) * (56 * u * np.abs(upd) + 30 * u * np.abs(wd * p)) + 1e-44
    if active is not None:
        new, err = np.where(active, new, p), np.where(active, err, 0.0)
    return new, err


def grad_norm(grads, max_norm=math.inf, unscale=1.0):
    total = math.fsum(float(np.sum(g.astype(np.float64) ** 2)) for g in grads)
    norm = unscale * math.sqrt(total) if math.isfinite(total) else math.nan
    scale = unscale * (1.0 if norm < max_norm else max_norm / norm) if math.isfinite(norm) else math.nan
    return norm, scale
