"""The 8-bit floating-point operators in numpy, in 64 bits, written from their definitions
in include/rembed_hip.h."""
import math

import numpy as np

BLOCK = 64

# every e4m3 code's value (0x7F and 0xFF are NaN)
CODES = np.array([math.nan if c & 127 == 127 else
                  (-1.0 if c & 128 else 1.0) *
                  ((c & 7) * 2.0 ** -9 if c >> 3 & 15 == 0
                   else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3 & 15) - 7)) for c in range(256)])


def exponent(top):
    """The byte x of the smallest 2^(x - 127) with top <= 448 * 2^(x - 127)."""
    m, e = np.frexp(np.asarray(top, np.float64) / 448)
    e = np.where(m == 0.5, e - 1, e) + 127
    return np.where(np.asarray(top) == 0, 0, np.clip(e, 0, 254)).astype(np.int64)


def encode(x):
    """Codes of the e4m3 values nearest to |x| <= 448, ties to even; NaN where x is none."""
    x = np.asarray(x, np.float64)
    a = np.abs(np.where(np.isfinite(x), x, 0.0))
    _, e = np.frexp(a)
    e = np.maximum(e - 1, -6)
    q = np.rint(a / 2.0 ** (e - 3.0))  # 8..16 of normal numbers
    code = np.where(q >= 8, (e + 7) * 8 + q - 8, q).astype(np.int64)  # 16 carries on
    code = code + 128 * np.signbit(x)
    return np.where(np.isfinite(x), code, 127).astype(np.uint8)


def two(x):
    return 2.0 ** (np.asarray(x, np.float64) - 127)


def quantize_rows(a):
    """[m][k] -> codes [m][kp], bytes [m][kp / 128], the values they stand for [m][k]."""
    m, k = a.shape
    kp = (k + 127) // 128 * 128
    x = np.zeros((m, kp))
    x[:, :k] = a
    x = x.reshape(m, -1, 128)
    top = np.where(np.isfinite(x), np.abs(x), 0).max(2)
    e = exponent(top)
    codes = encode(x / two(e)[:, :, None])
    vals = CODES[codes] * two(e)[:, :, None]
    return codes.reshape(m, kp), e, vals.reshape(m, kp)[:, :k]


def quantize_weight(w):
    """[n][k] -> codes [n][k], bytes [n][ceil(k/128)], values [n][k]."""
    n, k = w.shape
    x = np.zeros(((n + 127) // 128 * 128, (k + 127) // 128 * 128))
    x[:n, :k] = w
    b = x.reshape(x.shape[0] // 128, 128, -1, 128)
    e = exponent(np.abs(b).max((1, 3)))
    codes = encode(b / two(e)[:, None, :, None])
    vals = CODES[codes] * two(e)[:, None, :, None]
    return (codes.reshape(x.shape)[:n, :k], np.repeat(e, 128, 0)[:n],
            vals.reshape(x.shape)[:n, :k])


def scale_rows(sa, m, kb):
    """The scale bytes' layout undone: [m][kb]."""
    groups = (m + 127) // 128
    x = np.asarray(sa)[: groups * 128 * kb].reshape(kb, groups, 32, 4)
    return x.transpose(1, 3, 2, 0).reshape(groups * 128, kb)[:m]


# ---- the cache ----------------------------------------------------------------------

def k_at(t, d):
    return (((d // 64) * 2 + t // 32) * 2 + d % 32 // 16) * 1024 \
        + (d % 64 // 32 * 32 + t % 32) * 16 + d % 16


def v_at(t, d):
    return (d // 32 * 2 + t // 32) * 1024 + (t % 8 // 4 * 32 + d % 32) * 16 + t % 32 // 8 * 4 + t % 4


def places(at, dh):
    return at(np.arange(BLOCK)[:, None], np.arange(dh)[None])


class Cache:
    """Codes and bytes as the device holds them."""

    def __init__(self, pages, kv_heads, dh, fill=0x7F):
        self.pages, self.heads, self.dh = pages, kv_heads, dh
        self.k = np.full((pages, kv_heads, BLOCK * dh), fill, np.uint8)
        self.v = np.full((pages, kv_heads, BLOCK * dh), fill, np.uint8)
        self.k_exp = np.full((pages, kv_heads), 200, np.uint8)
        self.v_exp = np.full((pages, kv_heads), 200, np.uint8)

    def append(self, k, v, cu, slots):
        """k, v: [rows][heads][dh] float64; one request after another."""
        for b in range(len(cu) - 1):
            r = cu[b]
            while r < cu[b + 1]:
                off = int(slots[r] % BLOCK)
                n = min(BLOCK - off, cu[b + 1] - r)
                if 0 <= slots[r] < self.pages * BLOCK:
                    self._block(int(slots[r] // BLOCK), off, k[r:r + n], v[r:r + n])
                r += n

    def _block(self, page, off, k, v):
        for h in range(self.heads):
            bad = ~(np.isfinite(k[:, h]).all(1) & np.isfinite(v[:, h]).all(1))
            for x, codes, exps, at, is_k in ((k, self.k, self.k_exp, k_at, True),
                                             (v, self.v, self.v_exp, v_at, False)):
                y = np.where(bad[:, None], 0.0, x[:, h])
                e = int(exponent(np.abs(y).max()))
                where = places(at, self.dh)
                if off == 0:
                    kept = np.zeros((BLOCK, self.dh), np.uint8)
                else:
                    old = int(exps[page, h])
                    e = max(e, old)
                    kept = codes[page, h][where]
                    if e != old:
                        kept = encode(CODES[kept] * two(127 + old - e))
                kept[off:off + len(y)] = encode(y / two(e))
                if is_k:
                    kept[off:off + len(y)][bad] = 0x7F
                codes[page, h][where] = kept
                exps[page, h] = e

    def rows(self, table, n):
        """K and V of a request's first n tokens: [n][heads][dh]."""
        got = []
        for codes, exps, at in ((self.k, self.k_exp, k_at), (self.v, self.v_exp, v_at)):
            where = places(at, self.dh)
            x = np.empty((n, self.heads, self.dh))
            for j in range((n + BLOCK - 1) // BLOCK):
                c = min(BLOCK, n - j * BLOCK)
                for h in range(self.heads):
                    x[j * BLOCK:j * BLOCK + c, h] = (
                        CODES[codes[table[j], h][where[:c]]] * two(exps[table[j], h]))
            got.append(x)
        return got


def plan(past, fresh, free, table, rows):
    """cu, blocks, lens, slots, pos, status of rh_cache_plan; table is written on."""
    past, fresh = [int(x) for x in past], [int(x) for x in fresh]
    ldt = table.shape[1]
    err = 0
    if any(p < 0 or f < 0 for p, f in zip(past, fresh)):
        err |= 1
    ok = [(p, f) for p, f in zip(past, fresh) if p >= 0 and f >= 0]
    if any(-(-(p + f) // BLOCK) > ldt for p, f in ok):
        err |= 2
    if sum(f for _, f in ok) > rows:
        err |= 4
    if sum(-(-(p + f) // BLOCK) + -p // BLOCK for p, f in ok) > len(free):
        err |= 8
    n = len(past)
    cu, blocks = np.zeros(n + 1, np.int32), np.zeros(n + 1, np.int32)
    slots, pos = np.full(rows, -1, np.int64), np.zeros(rows, np.int32)
    if err:
        return cu, blocks, np.array(past, np.int32), slots, pos, [err, 0, 0, 0]
    taken = 0
    for b, (p, f) in enumerate(zip(past, fresh)):
        for j in range(-(-p // BLOCK), -(-(p + f) // BLOCK)):
            table[b, j] = free[taken]
            taken += 1
        at = cu[b]
        for t in range(f):
            page = int(table[b, (p + t) // BLOCK])
            slots[at + t] = -1 if page < 0 else page * BLOCK + (p + t) % BLOCK
            pos[at + t] = p + t
        cu[b + 1] = at + f
        blocks[b + 1] = blocks[b] + len({(p + t) // BLOCK for t in range(f)})
    return (cu, blocks, np.array(past, np.int32) + np.array(fresh, np.int32), slots, pos,
            [0, int(cu[n]), taken, int(blocks[n])])


def attention(q, k, v, scale, causal, window):
    """q [nq][heads][dh] at the last positions of k, v [n][kv][dh]. Also sum p |v| and the
    largest |q_i k_i| of a score, which the tolerances take."""
    nq, heads, dh = q.shape
    n, kv = k.shape[:2]
    out, mag = np.zeros_like(q), np.zeros_like(q)
    top = 0.0
    i = (n - nq + np.arange(nq))[:, None]
    j = np.arange(n)[None]
    see = np.ones((nq, n), bool)
    if causal:
        see &= j <= i
    if window:
        see &= np.abs(i - j) < window
    for h in range(heads):
        u = h // (heads // kv)
        kk, vv = k[:, u], v[:, u]
        s = np.where(see, (q[:, h] @ kk.T) * scale, -np.inf) if n else np.zeros((nq, 0))
        any_ = see.any(1)
        m = np.where(any_, s.max(1, initial=-np.inf), 0.0)
        with np.errstate(invalid="ignore"):
            p = np.exp(s - m[:, None])
        p = np.where(see, p, 0.0)
        total = p.sum(1, keepdims=True)
        p = np.divide(p, total, out=np.zeros_like(p), where=total != 0)
        with np.errstate(invalid="ignore"):
            out[:, h] = np.where(see[:, :, None], p[:, :, None] * vv[None], 0.0).sum(1) \
                if n * nq * dh <= 4_000_000 else p @ np.where(np.isnan(vv), 0, vv)
            mag[:, h] = p @ np.abs(vv)
        out[:, h] = np.where(any_[:, None], out[:, h], 0.0)
        if n and nq:
            top = max(top, np.nanmax(np.abs(q[:, h])) * np.nanmax(np.abs(kk)))
    return out, mag, top
