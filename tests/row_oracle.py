"""The row operators between a layer's products in numpy, in 64 bits, and how far fp32 may be off.

u = 2^-24 is half a step of fp32, relative to the value.
"""
import math

import numpy as np

import test_fp8_operators as F

U = 2.0 ** -24
# cos and sin of the kernels: the polynomials' rest 2e-9, the angle's roundings (2 u pi/4 at most), the
# fused steps, of which the last weighs most (u each), amp's product u
TURN = 2e-9 + 8 * U


def frequencies(rot, theta=10000.0, scaling=0, factor=1.0, original=0, fast=0.0, slow=0.0,
                freq=None):
    """Radians a position (longdouble) and amp; scaling as RH_ROPE_*."""
    one = np.longdouble(1)
    s, amp = one * factor, 1.0
    i = np.arange(rot // 2)
    if scaling == 5:
        return np.asarray(freq, np.longdouble), amp
    t = one * theta * (s ** (one * rot / (rot - 2)) if scaling == 2 else one)
    f = t ** (-2 * one * i / rot)
    if scaling == 1:
        f = f / s
    elif scaling == 3:
        at = [rot * math.log(original / (b * 2 * math.pi)) / (2 * math.log(theta))
              for b in (fast or 32, slow or 1)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        ramp = np.clip((i - lo) / ((hi - lo) or 0.001), 0, 1)
        f, amp = f * (1 - ramp) + f / s * ramp, 1 + 0.1 * math.log(factor)
    elif scaling == 4:
        a, b = slow or 1, fast or 4
        keep = np.clip((original * f / (2 * np.pi) - a) / (b - a), 0, 1)
        f = f * keep + f / s * (1 - keep)
    return f, amp


def cos_sin(pos, freq, amp):
    """[rows][1][pairs]; whole turns taken off in longdouble."""
    a = np.asarray(pos, np.longdouble)[:, None] * np.asarray(freq, np.longdouble)
    pi2 = 2 * np.arccos(np.longdouble(-1))
    a = (a - np.round(a / pi2) * pi2).astype(np.float64)[:, None]
    return amp * np.cos(a), amp * np.sin(a)


def head_norm(x, weight, eps):
    """RMS norm over the last axis, and how far fp32 may be off: a sum of dh squares in runs of
    at most 16 and then a tree of at most 6 (22 u, half of it in the root), root, quotient and two
    products."""
    inv = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    y = x * inv * (1.0 if weight is None else weight)
    return y, np.abs(y) * 18 * U


def turn(x, off, pos, freq, amp, halves):
    """x [rows][h][dh] turned, and how far off it may be where x is off by `off`."""
    n = len(freq)
    a, b = (np.arange(n), n + np.arange(n)) if halves else (2 * np.arange(n), 2 * np.arange(n) + 1)
    c, s = cos_sin(pos, freq, amp)
    y, far = x.copy(), off.copy()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    size = np.abs(x[..., a]) + np.abs(x[..., b])
    # the product that is rounded, the fused sum, cos and sin themselves
    far[..., a] = (off[..., a] * np.abs(c) + off[..., b] * np.abs(s)) + size * amp * (TURN + 3 * U)
    far[..., b] = (off[..., b] * np.abs(c) + off[..., a] * np.abs(s)) + size * amp * (TURN + 3 * U)
    return y, far


def stored(want, off, bf16):
    """How far a stored value may be off: its own rounding comes on top."""
    return off + (F.BF16 if bf16 else U) * (np.abs(want) + off) + 1e-37


def norm(x, off, kind, weight, bias, eps, n):
    """x [m][n] normed (kind as RH_NORM_*), and how far off where x is off by `off`. A thread adds at
    most 64 values, 8 more steps join the threads: 72 u of the sum of magnitudes."""
    if kind == 0:
        return x, off
    w = np.ones(n) if weight is None else weight
    b = np.zeros(n) if bias is None else bias
    d, od = x, off
    if kind == 2:
        d = x - x.mean(1, keepdims=True)
        od = off + off.mean(1, keepdims=True) + 74 * U * np.abs(x).mean(1, keepdims=True) + U * np.abs(d)
    ms = (d * d).mean(1, keepdims=True) + eps
    with np.errstate(divide="ignore", invalid="ignore"):
        inv = np.where(ms > 0, 1 / np.sqrt(ms), np.nan)
    # the mean square is off by 2 |d| od and od^2, and by its own sum
    rel = ((2 * np.abs(d) * od + od * od).mean(1, keepdims=True) / ms + 76 * U) / 2
    y = d * inv * w
    far = np.abs(w) * inv * (od + np.abs(d) * rel) * (1 + rel) + 6 * U * np.abs(y)
    return y + b, far + U * np.abs(y + b)


def residual(x, y, post, pre, gate, xs, ys):
    """sum and out, each with how far off; post and pre: (kind, weight, bias, eps)."""
    m, n = x.shape
    off = np.zeros((m, n))
    if y is None:
        s, off = xs * x, U * np.abs(xs * x)
    else:
        z, zo = norm(y, off, *post, n)
        g = np.ones(1) if gate is None else gate
        s = xs * x + ys * g * z
        off = np.abs(ys * g) * zo + 3 * U * np.abs(ys * g * z) + U * np.abs(s)
    out, far = norm(s, off, *pre, n)
    return s, off, out, far
