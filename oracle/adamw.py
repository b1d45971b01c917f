"""AdamW over separate tensors and the 8-bit form of its moments, on the CPU.

``step32`` repeats the kernels' float32 arithmetic operation by operation (its
moments are equal bit for bit); ``step64`` is the definition in 64 bits, with a
bound of what float32 arithmetic may add.  The 8-bit form is written from real
arithmetic (binades and multiples of a step), not from bit patterns.
"""
import numpy as np

BLOCK = 256
M_TOP, V_TOP = 15, 31
MIN_EXP = 64


def offsets_of(n, t, positive, first=0):
    """Rounding offsets in [0, 1) of elements first .. first + n at step t."""
    i = np.arange(first, first + n, dtype=np.uint64)
    w = (i * np.uint64(0x9E3779B1) + np.uint64(t) * np.uint64(0x6A09E667)) & np.uint64(0xFFFFFFFF)
    if positive:
        w = np.uint64(0xFFFFFFFF) - w
    return (w >> np.uint64(12)).astype(np.float64) / 2.0 ** 20


def quantize(x, t, positive, first=0):
    """(codes uint8 [padded], exponent bytes) of a flat float32 array."""
    top = V_TOP if positive else M_TOP
    n = x.size
    if n == 0:
        return np.zeros(0, np.uint8), np.zeros(0, np.uint8)
    room = -(-n // BLOCK) * BLOCK
    a = np.zeros(room)
    a[:n] = np.abs(x.astype(np.float64))
    bad = ~np.isfinite(a).reshape(-1, BLOCK).all(1)  # a value that is not finite takes its block with it
    a[np.repeat(bad, BLOCK)] = 0.0
    u = np.zeros(room)
    u[:n] = offsets_of(n, t, positive, first)
    own = np.exp2(np.frexp(np.maximum(a, 2.0 ** -126))[1] - 4.0)  # an eighth of x's binade
    most = (own * np.floor(a / own + u)).reshape(-1, BLOCK).max(1)
    field = np.where(most > 0, np.frexp(most)[1] + 126, 0)  # float32 exponent field
    field = np.clip(field, MIN_EXP, 255)
    e = np.repeat(field, BLOCK)
    low = np.exp2(e - (top - 1) - 127.0)  # smallest value with exponent field 1
    step = np.where(a < low, low / 8, own)
    k = np.floor(a / step + u)            # in steps; 8 .. 16 within a whole binade
    value = k * step
    f, b = np.frexp(value)                # value = f 2^b, f in [1/2, 1)
    whole = ((b + 126 - (e - top)) * 8 + (f * 16 - 8)).astype(np.int64)
    code = np.where(value < low, k.astype(np.int64), whole)
    if positive:
        code = np.where((a > 0) & (code == 0), 1, code)
    else:
        sign = np.zeros(room, np.int64)
        sign[:n] = np.signbit(x)
        code = code + 128 * sign
    field[bad] = 255
    assert code.min() >= 0 and code.max() <= 255
    return code.astype(np.uint8), field.astype(np.uint8)


def values(codes, exps, positive):
    """float32 values of codes (no number in a block whose exponent byte is 255)."""
    top = V_TOP if positive else M_TOP
    c = codes.astype(np.int64)
    sign = 1.0
    if not positive:
        sign = np.where(c >= 128, -1.0, 1.0)
        c = c & 127
    f, q = c >> 3, c & 7
    e = np.repeat(exps.astype(np.float64), BLOCK)
    mag = np.where(f == 0, q * 2.0 ** -2, (8 + q) * np.exp2(f - 3.0)) * np.exp2(e - 127.0 - top)
    return np.where(e == 255, np.nan, sign * mag).astype(np.float32)


def step32(g, m, v, *, beta1, beta2, scale=1.0):
    """New float32 moments, every operation rounded."""
    f = np.float32
    with np.errstate(all="ignore"):
        g = (g.astype(f) * f(scale)).astype(f)
        mn = f(beta1) * m + f(1.0 - beta1) * g
        vn = f(beta2) * v + f(1.0 - beta2) * (g * g)
    assert mn.dtype == f and vn.dtype == f
    return mn, vn


def step64(p, g, m, v, *, lr, beta1, beta2, eps, decay, t, scale=1.0):
    """(p, m, v, bound): the step in 64 bits and, per parameter, what float32
    arithmetic may add: with u = 2^-24, three roundings of p (factor, product,
    difference), at most sixteen relative ones of the step, four of them on m's
    two terms before they cancel."""
    p, g, m, v = (np.asarray(x, np.float64) for x in (p, g, m, v))
    g = g * scale
    a, b = beta1 * m, (1.0 - beta1) * g
    mn = a + b
    vn = beta2 * v + (1.0 - beta2) * g * g
    denom = np.sqrt(vn) / np.sqrt(1.0 - beta2 ** t) + eps
    rate = lr / (1.0 - beta1 ** t)
    d = rate * mn / denom
    pn = (1.0 - lr * decay) * p - d
    u = 2.0 ** -24
    bound = u * (3.0 * np.abs(p) + np.abs(pn) + 16.0 * np.abs(d) + 4.0 * rate * (np.abs(a) + np.abs(b)) / denom)
    return pn, mn, vn, bound
