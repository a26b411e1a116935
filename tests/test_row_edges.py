"""Edges of the row operators (residual norms, rotary rows, the rotary append, the cache read
back): one factor for a whole head, many heads at document sizes, what is refused, frequencies of
any size, codes next to a border. Against numpy in 64 bits (row_oracle, fp8_oracle).
"""
import ctypes

import numpy as np
import pytest

import fp8_oracle as O
import row_oracle as R
import test_fp8_operators as F

I32 = np.int32


# ---- a norm that is none -------------------------------------------------------------------

def at(p):
    return ctypes.c_void_p(p)


def passes(fn, *args):
    """The call's checks let it through as far as to the context, which there is none."""
    from rembed_amd import _lib as L
    F.refused(L.RH_ERR_INVALID, fn, None, *args)
    assert b"null context" in L.lib.rh_last_error(), L.lib.rh_last_error()


def test_a_norm_that_is_none_names_no_memory():
    from rembed_amd import _lib as L
    rows = [at(1 << 20), 0, 256, at(2 << 20), 0, 256, at(3 << 20), 256, at(4 << 20), 1, 256, None, 0, None,
            9, 256, None]
    stale = L.NormDesc(0, float("nan"), 3 << 20, 1 + (4 << 20))  # on the outputs, and at odd bytes
    none = L.NormDesc()
    for post, pre in ((stale, none), (none, stale), (stale, stale)):
        passes("rh_residual_norm", L.ResidualDesc(post, pre, None, 0, 1.0, 1.0), *rows)
    rows[3] = None                                               # no y: a post norm of a kind is refused
    passes("rh_residual_norm", L.ResidualDesc(stale, none, None, 0, 1.0, 1.0), *rows)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1024, 1001, 16384])
def test_a_norm_that_is_none_is_not_read(gpu_ctx, n):
    """Weights of NaN that a norm of no kind names, at bytes that no 16-byte load takes: the bits
    of null ones."""
    from rembed_amd import _lib as L
    from rembed_amd import tensor as T
    rng = np.random.default_rng(n)
    m = 5
    x, y = (gpu_ctx.upload(rng.standard_normal((m, n)).astype(np.float32)) for _ in "xy")
    nan = gpu_ctx.upload(np.full(n + 1, np.nan, np.float32))
    got = []
    for w in (None, nan.ptr + 4):
        out, total = gpu_ctx.alloc(m * n * 4), gpu_ctx.alloc(m * n * 4)
        res = T.Residual()
        for norm in (res.desc.post, res.desc.pre):
            norm.kind, norm.eps, norm.weight, norm.bias = L.RH_NORM_NONE, 1e-6, w, w
        T.ResidualNorm(gpu_ctx, res, x, False, n, y, False, n, total, n, out, False, n, None, 0, None, m, n)
        gpu_ctx.sync()
        got.append([b.download(np.uint32, (m, n)) for b in (out, total)])
    for a, b in zip(*got):
        assert np.array_equal(a, b) and np.isfinite(a.view(np.float32)).all()


# ---- GPU: frequencies of any size ------------------------------------------------------------

BITS = 1400


def machin():
    """pi * 2^BITS in whole numbers: 16 arctan(1/5) - 4 arctan(1/239)."""
    def arctan(n):
        x = (1 << BITS) // n
        total, i = 0, 1
        while x:
            total += x // i if i % 4 == 1 else -(x // i)
            x //= n * n
            i += 2
        return total
    return 16 * arctan(5) - 4 * arctan(239)


def turn_fraction(pos, freq, pi):
    """pos * freq / (2 pi) less the nearest whole number, within 2^-63."""
    n, d = float(freq).as_integer_ratio()
    u = (pos * n << BITS + 64) // (2 * d * pi) % (1 << 64)
    return (u - (1 << 64) if u >> 63 else u) / 2.0 ** 64


@pytest.mark.gpu
def test_rope_of_given_frequencies_of_any_size(gpu_ctx):
    """Angles within 2^-31 of a turn at every position: a sine near a whole turn shows them. Sine and
    cosine are those of pi from whole numbers."""
    from rembed_amd import tensor as T
    rng = np.random.default_rng(0)
    pi = machin()
    assert abs(pi / (1 << BITS) - np.pi) < 1e-15
    freq = [0.0, 5e-324, 1e-30, 2.0 ** -40, 0.37, 1.0, np.pi, 2 * np.pi, 50.0, -50.0, 1e3, -12345.678, 1e6, 2.0 ** 53,
            1e16, -3e18, 2.0 ** 63, 2.0 ** 64, 1e20, -1e25, 1e30, 1.7e38, 2.0 ** 127, 1e50, -1e77, 1e100, 1e150, 2.0 ** 640,
            1e200, -1e250, 1e300, np.finfo(np.float64).max]
    n, dh = len(freq), 2 * len(freq)
    pos = np.concatenate([[0, 1, -1, 2, 2 ** 31 - 1, -2 ** 31], rng.integers(-2 ** 31, 2 ** 31, 2000)])
    # those whose angle of one of the frequencies is next to a whole turn, and some others
    frac = np.array([[turn_fraction(int(p), f, pi) for f in freq] for p in pos])
    pick = np.unique(np.concatenate([np.arange(60), np.abs(np.where(frac == 0, 1, frac)).argmin(0)]))
    pos, frac = pos[pick].astype(I32), frac[pick]
    x = np.zeros((len(pos), dh), np.float32)
    x[:, :n] = 1.0                                 # (1, 0) becomes (cos, sin)
    rope = T.Rope(gpu_ctx, dh, scaling=5, freq=freq)
    out = gpu_ctx.alloc(x.nbytes)
    T.RopeRows(gpu_ctx, rope, gpu_ctx.upload(x), False, dh, out, False, dh, 0, 0, -1, 1, 0, dh,
               gpu_ctx.upload(pos), len(pos))
    gpu_ctx.sync()
    got = out.download(np.float32, x.shape).astype(np.float64)
    c, s = np.cos(2 * np.pi * frac), np.sin(2 * np.pi * frac)
    off = 2 * np.pi * 2.0 ** -31
    # relative where the sine is small: its polynomial, t itself and two products round it
    assert (np.abs(got[:, n:] - s) <= off + R.TURN * np.abs(s)).all()
    assert (np.abs(got[:, :n] - c) <= off * np.abs(s) + off ** 2 + R.TURN).all()


# ---- GPU: the rotary append's norm of K ---------------------------------------------------

def cached_k(ctx, rope, norm, x, kv, dh):
    """K rows [n][kv][dh] (fp32, v zeros), a request and page each, at position 0, through the
    rotary append: the codes [n][kv][dh]."""
    from rembed_amd import tensor as T
    n = x.shape[0]
    rows = np.concatenate([x.reshape(n, -1), np.zeros((n, kv * dh))], 1).astype(np.float32)
    cu, blk, _, slots, pos, _ = O.plan([0] * n, [1] * n, list(range(n)), np.zeros((n, 1), I32), n)
    c = O.Cache(n, kv, dh)
    dev = F.device_cache(ctx, c)
    T.RopeAppend(ctx, rope, dev, ctx.upload(rows), False, rows.shape[1], 0, 0, kv * dh, None, False, 0,
                 0, ctx.upload(pos), ctx.upload(cu), ctx.upload(blk), ctx.upload(slots), n, n, None, norm)
    ctx.sync()
    k = dev.k.download(np.uint8, c.k.shape)
    return k[:, :, O.places(O.k_at, dh)[0]]


@pytest.mark.gpu
@pytest.mark.parametrize("dh,kv,parts", [(64, 1, 4), (128, 2, 4), (128, 1, 8), (256, 1, 8)])
def test_rope_append_norms_a_head_by_one_factor(gpu_ctx, dh, kv, parts):
    """Equal values of a head have equal codes, whichever of the token's threads has them. The values
    stand within four steps of fp32 of the place where their normed values change codes, so that
    factors a step apart give other codes."""
    from rembed_amd import tensor as T
    rng = np.random.default_rng(dh + parts)
    n = 300                       # 300 blocks of two heads are over 512 workgroups: four threads a token
    x = rng.standard_normal((n, kv, dh)).astype(np.float32).astype(np.float64)
    at = 8 * np.arange(parts)[:, None] + np.arange(8)  # eight values of each thread
    x[..., at] = 0
    border = 0.53125              # between the codes 0.5 and 0.5625, and 2^-k of them
    mean = (x * x).sum(-1) / dh / (1 - 8 * parts * border ** 2 / dh)
    near = (border * np.sqrt(mean + 1e-6)).astype(np.float32)
    steps = np.arange(-4, 4)
    x[..., at] = (near.view(I32)[..., None] + steps).astype(I32).view(np.float32)[:, :, None]
    codes = cached_k(gpu_ctx, T.Rope(gpu_ctx, dh), T.Norm(None, 1e-6), x, kv, dh)[..., at]
    assert (codes == codes[:, :, :1]).all()
    below = (codes[:, :, 0, 0] != codes[:, :, 0, 7]).mean()
    assert below > 0.5            # the border is among them
