"""CPU restatements of the 8-bit linear layers in whole numbers (numpy int64, Python integers where
they pass 64 bits).  TEST INFRASTRUCTURE ONLY (the oracle, never the thing measured or shipped).
Nothing here imports the product."""
from fractions import Fraction

import numpy as np


def quant(x):
    """(codes [n][k], maxima [n]) of int16 rows."""
    x = np.asarray(x, np.int64)
    a = np.abs(x).max(axis=1)
    r = np.where(a > 0, (127 * 2 ** 24 + a // 2) // np.maximum(a, 1), 0)
    return (x * r[:, None] + 2 ** 23) >> 24, a


def rne_ratio(num, den):
    """The whole number next to num / den (den > 0), ties to the even one."""
    q, r = divmod(num, den)
    return q + (1 if 2 * r > den or (2 * r == den and q & 1) else 0)


def sums(codes, w):
    """sum_k c w: whole numbers below 2^53, so float64's BLAS is exact."""
    return (np.asarray(codes, np.float64) @ np.asarray(w, np.float64)).astype(np.int64)


def scaled(acc, a, mult, bias=None):
    """sat16(rne(acc a mu + b)) exactly: the multipliers as ratios of integers."""
    n, m = acc.shape
    out = np.zeros((n, m), np.int64)
    for j in range(m):
        f = Fraction(float(mult[j]))
        num, den, b = f.numerator, f.denominator, 0 if bias is None else int(bias[j])
        for t in range(n):
            out[t, j] = rne_ratio(int(acc[t, j]) * int(a[t]) * num + b * den, den)
    return np.clip(out, -32768, 32767)


def scaled_fast(acc, a, mult, bias=None):
    """scaled for multipliers M 2^-s of at most 18 bits and sums below 2^62, in int64."""
    man, exp = np.frexp(np.asarray(mult, np.float64))
    M, s = np.rint(man * 2.0 ** 18).astype(np.int64), 18 - exp.astype(np.int64)
    assert (np.ldexp(M.astype(np.float64), -s) == mult).all() and (s >= 1).all() and (s < 62).all()
    y = acc * a[:, None] * M
    if bias is not None:
        y = y + (np.asarray(bias, np.int64) << s)
    q = y >> s
    rem, half = y - (q << s), np.int64(1) << (s - 1)
    return np.clip(q + ((rem > half) | ((rem == half) & (q & 1 == 1))), -32768, 32767)


def linear(x, w, mult, bias=None, residual=None, shift=0, exact=False):
    codes, a = quant(x)
    o = (scaled if exact else scaled_fast)(sums(codes, w), a, mult, bias)
    if residual is None:
        return o.astype(np.int16)
    return np.clip(np.asarray(residual, np.int64) + (o << shift), -2 ** 31, 2 ** 31 - 1).astype(np.int32)


def sigmoid_pieces():
    return np.rint(2.0 ** 24 / (1.0 + np.exp(-np.arange(4097) / 256.0))).astype(np.int64)


def gate(g, u, act, gate_shift, out_shift, act_table=None):
    """act(g) u 2^-out_shift; act_table the activation unit's [65536] (oracle.cm.act_table) for the GELUs."""
    g, u = np.asarray(g, np.int64), np.asarray(u, np.int64)
    if act == "silu":
        T, gv = sigmoid_pieces(), g << gate_shift
        at = np.minimum(np.abs(gv), (16 << 14) - 1)
        sig = T[at >> 6] + (((T[(at >> 6) + 1] - T[at >> 6]) * (at & 63)) >> 6)
        sig = np.where(np.abs(gv) >= 16 << 14, 1 << 24, sig)
        f = _rne(gv * np.where(gv < 0, (1 << 24) - sig, sig), 18)
    else:
        f = np.asarray(act_table, np.int64)[g + 32768]
    return np.clip(_rne(f * u, out_shift), -32768, 32767)


def _rne(x, e):
    if e == 0:
        return x
    q = x >> e
    rem, half = x - (q << e), 1 << (e - 1)
    return q + ((rem > half) | ((rem == half) & (q & 1 == 1)))


def gated(x, wg, wu, mg, mu, act, gate_shift, out_shift, act_table=None, bg=None, bu=None, exact=False):
    codes, a = quant(x)
    f = scaled if exact else scaled_fast
    g, u = f(sums(codes, wg), a, mg, bg), f(sums(codes, wu), a, mu, bu)
    return gate(g, u, act, gate_shift, out_shift, act_table).astype(np.int16)
