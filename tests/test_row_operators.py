"""Residual norms, rotary rows, the rotary append and the cache read back, against numpy in 64 bits
(row_oracle, fp8_oracle). Tolerances count roundings: row_oracle derives them from the sums'
lengths, and a stored value adds half a step of its type.
"""
import ctypes

import numpy as np
import pytest

import fp8_oracle as O
import row_oracle as R
import test_fp8_operators as F

I32 = np.int32


# ---- CPU: frequencies, refusals ---------------------------------------------------------

SCALINGS = [dict(), dict(theta=1e6), dict(scaling=1, factor=4.0), dict(scaling=2, factor=8.0),
            dict(scaling=3, factor=4.0, original=8192), dict(scaling=3, factor=40.0, original=100,
                                                             fast=8.0, slow=2.0),
            dict(scaling=4, factor=8.0, original=8192), dict(scaling=4, factor=2.0, original=64,
                                                             fast=6.0, slow=3.0)]


@pytest.mark.parametrize("rot", [4, 10, 64, 128, 256])
@pytest.mark.parametrize("kw", SCALINGS, ids=str)
def test_rope_frequencies(rot, kw):
    from rembed_amd import tensor as T
    f, amp = T.rope_frequencies(rot, **kw)
    want, a = R.frequencies(rot, **kw)
    # powers, logarithms and means in 64 bits and more: a few roundings of 2^-53
    assert np.allclose(f, want.astype(np.float64), rtol=1e-13, atol=0) and abs(amp - a) < 1e-15
    assert T.rope_frequencies(rot, amp=0.7, **kw)[1] == 0.7
    if not kw:
        assert f[0] == 1.0 and abs(f[-1] - 10000.0 ** (2.0 / rot - 1)) < 1e-15


def test_rope_frequencies_all_fast_or_all_slow():
    """YaRN where every pair turns over `fast` times, or under `slow`: none, all are scaled."""
    from rembed_amd import tensor as T
    plain, _ = T.rope_frequencies(16, theta=1.5)
    same, _ = T.rope_frequencies(16, theta=1.5, scaling=3, factor=8.0, original=1 << 30)
    assert np.array_equal(same, plain)
    all_, _ = T.rope_frequencies(16, theta=1.5, scaling=3, factor=8.0, original=1)
    assert np.allclose(all_, plain / 8, rtol=1e-15)


def test_rope_frequencies_given():
    from rembed_amd import _lib as L
    from rembed_amd import tensor as T
    f, amp = T.rope_frequencies(6, scaling=5, freq=[0.5, -3.0, 100.0])
    assert f.tolist() == [0.5, -3.0, 100.0] and amp == 1.0
    with pytest.raises(L.RembedError):
        T.rope_frequencies(6, scaling=5, freq=[1.0])


def test_rope_config_refusals():
    from rembed_amd import _lib as L

    def no(code, **kw):
        c = L.RopeConfig(0, 64, 0, 0, 10000.0, 1.0, 0.0, 0.0, 0.0, None)
        for k, v in kw.items():
            setattr(c, k, v)
        F.refused(code, "rh_rope_frequencies", c, None, None)
        h = ctypes.c_void_p()
        F.refused(code, "rh_rope_create", None, c, ctypes.byref(h))

    F.refused(L.RH_ERR_INVALID, "rh_rope_frequencies", None, None, None)
    nan, inf = float("nan"), float("inf")
    for layout in (-1, 2):
        no(L.RH_ERR_INVALID, layout=layout)
    for rot in (0, -2, 3, 258):
        no(L.RH_ERR_SHAPE, rot=rot)
    for scaling in (-1, 6):
        no(L.RH_ERR_INVALID, scaling=scaling)
    for theta in (1.0, 0.0, -5.0, nan, inf):
        no(L.RH_ERR_INVALID, theta=theta)
    for factor in (0.5, 0.0, nan, inf):
        no(L.RH_ERR_INVALID, factor=factor, scaling=1)
    for amp in (-1.0, nan, inf):
        no(L.RH_ERR_INVALID, amp=amp)
    no(L.RH_ERR_SHAPE, scaling=2, rot=2)
    for scaling in (3, 4):
        no(L.RH_ERR_INVALID, scaling=scaling, original=0)
        for fast, slow in ((1.0, 2.0), (2.0, 2.0), (4.0, -1.0), (inf, 1.0), (nan, 1.0), (4.0, nan)):
            no(L.RH_ERR_INVALID, scaling=scaling, original=64, fast=fast, slow=slow)
    no(L.RH_ERR_INVALID, scaling=5)
    bad = (ctypes.c_double * 32)(*([0.0] * 31 + [nan]))
    no(L.RH_ERR_NONFINITE, scaling=5, freq=ctypes.addressof(bad))
    ok = L.RopeConfig(0, 64, 0, 0, 10000.0, 1.0, 0.0, 0.0, 0.0, None)
    F.refused(L.RH_ERR_INVALID, "rh_rope_create", None, ok, None)
    h = ctypes.c_void_p()
    F.refused(L.RH_ERR_INVALID, "rh_rope_create", None, ok, ctypes.byref(h))  # no context
    L.lib.rh_rope_destroy(None)


def at(p):
    return ctypes.c_void_p(p)


def test_residual_refusals():
    from rembed_amd import _lib as L
    none, rms = L.NormDesc(), L.NormDesc(1, 1e-6, None, None)
    base = dict(post=none, pre=rms, gate=None, ldg=0, x_scale=1.0, y_scale=1.0)
    # far apart: x, y, sum, out, codes, scales
    ok = [None, None, at(1 << 20), 0, 256, at(2 << 20), 0, 256, at(3 << 20), 256, at(4 << 20), 1, 256,
          at(5 << 20), 256, at(6 << 20), 9, 256, None]

    def no(code, res=None, **kw):
        a = list(ok)
        a[1] = L.ResidualDesc(**{**base, **(res or {})})
        for i, v in kw.items():
            a[int(i[1:])] = v
        F.refused(code, "rh_residual_norm", *a)

    no(L.RH_ERR_INVALID)                                          # no context
    F.refused(L.RH_ERR_INVALID, "rh_residual_norm", *ok)          # no residual
    no(L.RH_ERR_INVALID, a16=-1)
    no(L.RH_ERR_INVALID, a17=0)
    no(L.RH_ERR_SHAPE, a17=16385, a4=16385, a7=16385, a9=16385, a12=16385, a14=16512)
    no(L.RH_ERR_INVALID, dict(pre=L.NormDesc(3, 0, None, None)))
    no(L.RH_ERR_INVALID, dict(post=L.NormDesc(-1, 0, None, None)))
    for eps in (-1e-6, float("nan"), float("inf")):
        no(L.RH_ERR_INVALID, dict(pre=L.NormDesc(1, eps, None, None)))
    no(L.RH_ERR_INVALID, dict(pre=L.NormDesc(1, 0, None, 4096)))  # RMS with a bias
    no(L.RH_ERR_INVALID, dict(pre=L.NormDesc(2, 0, 4098, None)))
    for s in ("x_scale", "y_scale"):
        no(L.RH_ERR_INVALID, {s: float("inf")})
    no(L.RH_ERR_INVALID, dict(post=rms), a5=None)                 # a norm of nothing
    no(L.RH_ERR_INVALID, dict(gate=4096), a5=None)
    no(L.RH_ERR_SHAPE, dict(gate=4096, ldg=255))
    no(L.RH_ERR_SHAPE, dict(gate=4096, ldg=-1))
    no(L.RH_ERR_INVALID, dict(gate=4097))
    no(L.RH_ERR_INVALID, a8=None, a10=None, a13=None, a15=None)   # nothing to write
    no(L.RH_ERR_INVALID, a15=None)
    no(L.RH_ERR_INVALID, a13=None)
    no(L.RH_ERR_INVALID, a2=None)
    for i in (4, 7, 9, 12):
        no(L.RH_ERR_SHAPE, **{"a%d" % i: 255})
    no(L.RH_ERR_SHAPE, a14=384)
    for i, p in ((2, 2), (5, 2), (8, 2), (10, 1), (13, 8), (15, 2), (18, 2)):
        no(L.RH_ERR_INVALID, **{"a%d" % i: at((7 << 20) + p)})
    # overlaps: shifted, of another type, of another stride, outputs on each other
    no(L.RH_ERR_INVALID, a8=at((1 << 20) + 4))
    no(L.RH_ERR_INVALID, a8=at(1 << 20), a9=260)
    no(L.RH_ERR_INVALID, a10=at(1 << 20))                         # bf16 out on fp32 x
    no(L.RH_ERR_INVALID, a10=at(3 << 20), a11=0)                  # out on sum
    no(L.RH_ERR_INVALID, a13=at(1 << 20))
    no(L.RH_ERR_INVALID, a15=at((1 << 20) + 1024))
    no(L.RH_ERR_INVALID, a15=at((5 << 20) + 256))
    no(L.RH_ERR_INVALID, dict(gate=3 << 20, ldg=256))
    no(L.RH_ERR_INVALID, dict(gate=(3 << 20) + 1024))
    no(L.RH_ERR_INVALID, dict(pre=L.NormDesc(1, 0, (4 << 20) + 512, None)))
    no(L.RH_ERR_INVALID, dict(pre=L.NormDesc(2, 0, None, 5 << 20)))
    no(L.RH_ERR_INVALID, dict(post=L.NormDesc(1, 0, 6 << 20, None)))


def test_rotary_refusals_without_a_handle():
    from rembed_amd import _lib as L
    P = F.P
    rows = [None, None, P, 1, 512, at(1 << 20), 1, 512, 0, 256, -1, 4, 2, 64, P, 5, None, None, None]
    F.refused(L.RH_ERR_INVALID, "rh_rope_rows", *rows)
    for i, v, code in ((15, -1, L.RH_ERR_INVALID), (11, -1, L.RH_ERR_INVALID),
                       (12, -1, L.RH_ERR_INVALID), (13, 63, L.RH_ERR_SHAPE),
                       (13, 0, L.RH_ERR_SHAPE), (13, 258, L.RH_ERR_SHAPE)):
        a = list(rows)
        a[i] = v
        F.refused(code, "rh_rope_rows", *a)
    app = [None, None, F.desc(), P, 1, 512, 0, 256, 384, at(1 << 20), 1, 256, 4, P, P, P, P, 2, 9,
           None, None]
    F.refused(L.RH_ERR_INVALID, "rh_rope_append", *app)
    for i, v, code in ((2, None, L.RH_ERR_INVALID), (2, F.desc(dh=32), L.RH_ERR_SHAPE),
                       (12, -1, L.RH_ERR_INVALID), (17, -1, L.RH_ERR_INVALID),
                       (18, -1, L.RH_ERR_INVALID)):
        a = list(app)
        a[i] = v
        F.refused(code, "rh_rope_append", *a)


def test_read_refusals():
    from rembed_amd import _lib as L
    P = F.P
    ok = [None, F.desc(), P, 4, P, None, 2, 9, at(1 << 20), 1, 256, 0, 128]

    def no(code, **kw):
        a = list(ok)
        for i, v in kw.items():
            a[int(i[1:])] = v
        F.refused(code, "rh_cache_read", *a)

    no(L.RH_ERR_INVALID)
    no(L.RH_ERR_INVALID, a1=None)
    no(L.RH_ERR_SHAPE, a1=F.desc(dh=96))
    no(L.RH_ERR_INVALID, a6=-1)
    no(L.RH_ERR_INVALID, a7=-1)
    no(L.RH_ERR_SHAPE, a3=0)
    for i in (2, 4, 8):
        no(L.RH_ERR_INVALID, **{"a%d" % i: None})
    no(L.RH_ERR_SHAPE, a11=-8)
    no(L.RH_ERR_SHAPE, a12=136)
    no(L.RH_ERR_SHAPE, a12=120)                    # K and V share columns
    no(L.RH_ERR_SHAPE, a10=260)
    no(L.RH_ERR_SHAPE, a11=4, a10=264, a12=136)
    no(L.RH_ERR_SHAPE, a8=at((1 << 20) + 8))
    no(L.RH_ERR_SHAPE, a6=1 << 22)
    no(L.RH_ERR_SHAPE, a7=1 << 29, a6=0, a1=F.desc(heads=2))


# ---- GPU: helpers -----------------------------------------------------------------------

class At:
    """A place in a device buffer."""

    def __init__(self, buf, byte):
        self.buf, self.ptr = buf, buf.ptr + byte


def marked(ctx, rows, ld, bf16):
    """Rows full of a mark, and what reads them: values, and the marks that are left."""
    buf = ctx.upload(np.full((max(rows, 1), ld), 0x4242, np.uint16) if bf16
                     else np.full((max(rows, 1), ld), 55, np.float32))

    def read():
        ctx.sync()
        if bf16:
            bits = buf.download(np.uint16, (rows, ld))
            return F.from_bf16(bits), bits == 0x4242
        got = buf.download(np.float32, (rows, ld))
        return got, got == 55

    return buf, read


# ---- GPU: rotary rows -------------------------------------------------------------------

ROPE = [  # rows, heads, kv, dh, rot, layout, columns before / behind / more in out
    (1, 1, 0, 2, 2, 0, 0, 0, 0), (1, 16, 8, 128, 128, 0, 0, 0, 0), (5, 3, 1, 256, 256, 0, 8, 8, 0),
    (3, 2, 2, 64, 32, 1, 0, 0, 8), (7, 1, 1, 32, 32, 1, 16, 0, 0), (130, 12, 12, 64, 64, 1, 0, 8, 8),
    (33, 4, 1, 128, 32, 0, 0, 0, 0), (9, 2, 1, 256, 64, 1, 0, 0, 0), (4, 5, 0, 96, 96, 0, 0, 0, 0),
    (6, 0, 3, 64, 64, 0, 8, 0, 0), (11, 2, 1, 80, 20, 1, 3, 1, 2), (10, 3, 3, 128, 128, 0, 1, 0, 0),
    (8, 2, 2, 254, 250, 0, 0, 0, 0), (12, 1, 2, 64, 2, 1, 0, 0, 0), (2, 40, 20, 128, 128, 1, 0, 0, 0),
    (1100, 2, 1, 64, 64, 0, 0, 0, 0), (2, 1, 1, 32, 24, 0, 0, 0, 0), (3, 300, 8, 32, 32, 0, 0, 0, 0),
    (700, 6, 1, 256, 128, 0, 0, 0, 0), (2, 2, 1, 128, 100, 0, 0, 0, 4),
    # neighbours in runs of 2 and 4 of which one half turns in part, halves of an odd number of pairs
    (5, 2, 1, 128, 14, 1, 0, 0, 0), (9, 2, 2, 128, 68, 1, 8, 0, 0), (4, 2, 1, 36, 18, 1, 2, 0, 0),
    (700, 4, 1, 36, 18, 0, 0, 0, 0), (700, 4, 2, 200, 120, 0, 4, 0, 0), (900, 4, 1, 96, 50, 1, 0, 0, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16"),
                                       ("bf16", "f32")])
@pytest.mark.parametrize("i", range(len(ROPE)), ids=lambda i: "%d-%dx%d-%d-%d-%d" % ROPE[i][:6])
def test_rope_rows(gpu_ctx, i, dtype, out):
    from rembed_amd import tensor as T
    rows, heads, kv, dh, rot, layout, front, back, wider = ROPE[i]
    rng = np.random.default_rng(i)
    normed, values = i % 3 != 1, i % 2 == 0 and kv > 0
    kw = SCALINGS[i % len(SCALINGS)] if rot > 2 else {}
    width = (heads + 2 * kv) * dh
    x = rng.standard_normal((rows, front + width + back)) * np.exp(rng.uniform(-3, 3, (rows, 1)))
    img, val = F.typed(x, dtype)
    val = val.astype(np.float64)[:, front:front + width].reshape(rows, -1, dh)
    pos = rng.integers(0, 200000, rows).astype(I32)
    pos[0] = 0 if i % 2 else 5
    w = [rng.uniform(0.5, 1.5, dh).astype(np.float32) for _ in "qk"]
    d = [gpu_ctx.upload(a) for a in w]
    norms = [T.Norm(d[0], 1e-6), T.Norm(d[1], 1e-3)] if normed else [None, None]
    rope = T.Rope(gpu_ctx, rot, layout=layout, **kw)
    ld = front + width + back + wider
    buf, read = marked(gpu_ctx, rows + 2, ld, out == "bf16")
    off = [front, front + heads * dh, front + (heads + kv) * dh]
    T.RopeRows(gpu_ctx, rope, gpu_ctx.upload(img), dtype == "bf16", x.shape[1], buf, out == "bf16", ld,
               off[0], off[1], off[2] if values else -1, heads, kv, dh, gpu_ctx.upload(pos), rows,
               *norms)
    got, left = read()
    end = off[2] + (kv * dh if values else 0)
    assert left[rows:].all() and left[:, :front].all() and left[:, end:].all()
    got = got[:rows, front:end].reshape(rows, -1, dh)
    check_heads(got, val, heads, kv, dh, rot, layout, kw, pos, w if normed else None, out == "bf16")
    if values:
        want = val[:, heads + kv:]
        tol = F.BF16 * np.abs(want) if out == "bf16" and dtype == "f32" else 0
        assert (np.abs(got[:, heads + kv:] - want) <= tol).all()


def check_heads(got, val, heads, kv, dh, rot, layout, kw, pos, w, bf16, eps=(1e-6, 1e-3)):
    freq, amp = R.frequencies(rot, **kw)
    for part, cols in enumerate((slice(0, heads), slice(heads, heads + kv))):
        y, off = val[:, cols], np.zeros_like(val[:, cols])
        if w is not None:
            y, off = R.head_norm(y, w[part], eps[part])
        y, off = R.turn(y, off, pos, freq, amp, layout == 0)
        assert (np.abs(got[:, cols] - y) <= R.stored(y, off, bf16)).all(), part


@pytest.mark.gpu
def test_rope_rows_in_place(gpu_ctx):
    """On x itself: the bits of another buffer's, v and everything else left."""
    from rembed_amd import tensor as T
    rng = np.random.default_rng(1)
    for dtype, dh, rot, front in (("bf16", 128, 128, 8), ("f32", 64, 32, 0), ("bf16", 80, 80, 1)):
        width = 7 * dh + front
        img, _ = F.typed(rng.standard_normal((37, width)), dtype)
        pos = gpu_ctx.upload(rng.integers(0, 9999, 37).astype(I32))
        rope, n = T.Rope(gpu_ctx, rot, layout=1), T.Norm(None, 1e-6)
        x, out = gpu_ctx.upload(img), gpu_ctx.upload(img)
        bf = dtype == "bf16"
        args = (front, front + 4 * dh, -1, 4, 1, dh, pos, 37, n, n)
        T.RopeRows(gpu_ctx, rope, x, bf, width, out, bf, width, *args)
        T.RopeRows(gpu_ctx, rope, x, bf, width, x, bf, width, *args)
        args = args[:2] + (front + 5 * dh,) + args[3:]
        y = gpu_ctx.upload(img)
        T.RopeRows(gpu_ctx, rope, y, bf, width, y, bf, width, *args)  # v is where it is to go
        gpu_ctx.sync()
        a, b, c = (z.download(img.dtype, img.shape) for z in (x, out, y))
        assert np.array_equal(a, b) and np.array_equal(a, c) and not np.array_equal(a, img)
        assert np.array_equal(a[:, front + 5 * dh:], img[:, front + 5 * dh:])


@pytest.mark.gpu
def test_rope_rows_far_and_backwards(gpu_ctx):
    """Positions to the ends of 32 bits; a turn by p and one by -p give the input back."""
    from rembed_amd import tensor as T
    rng = np.random.default_rng(2)
    pos = np.array([0, 1, -1, 65536, 10 ** 6 + 1, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31, -12345], I32)
    n, dh = len(pos), 128
    x = rng.standard_normal((n, 2 * dh)).astype(np.float32)
    given = rng.uniform(-50, 50, dh // 2)
    for kw in (dict(), dict(scaling=5, freq=given)):
        for layout in (0, 1):
            rope = T.Rope(gpu_ctx, dh, layout=layout, **kw)
            y, z = gpu_ctx.alloc(x.nbytes), gpu_ctx.alloc(x.nbytes)
            d = gpu_ctx.upload(x)
            T.RopeRows(gpu_ctx, rope, d, False, 2 * dh, y, False, 2 * dh, 0, dh, -1, 1, 1, dh,
                       gpu_ctx.upload(pos), n)
            back = np.where(pos == -2 ** 31, pos, -pos).astype(I32)
            T.RopeRows(gpu_ctx, rope, y, False, 2 * dh, z, False, 2 * dh, 0, dh, -1, 1, 1, dh,
                       gpu_ctx.upload(back), n)
            gpu_ctx.sync()
            val = x.astype(np.float64).reshape(n, 2, dh)
            got = y.download(np.float32, x.shape).reshape(n, 2, dh)
            check_heads(got, val, 1, 1, dh, dh, layout, kw, pos, None, False)
            ok = pos != -2 ** 31
            again = z.download(np.float32, x.shape).reshape(n, 2, dh)[ok]
            assert np.abs(again - val[ok]).max() <= 8 * (R.TURN + 4 * R.U) * np.abs(val).max()


@pytest.mark.gpu
@pytest.mark.parametrize("dh", [64, 80])
def test_rope_rows_used(gpu_ctx, dh):
    """Rows from the device's count on are left; a count below 0 or above rows."""
    from rembed_amd import tensor as T
    x = np.ones((70, 2 * dh), np.float32)
    rope, pos = T.Rope(gpu_ctx, dh), gpu_ctx.upload(np.arange(70, dtype=I32))
    for used, done in ((0, 0), (1, 1), (69, 69), (70, 70), (1000, 70), (-3, 0)):
        buf, read = marked(gpu_ctx, 72, 2 * dh, False)
        T.RopeRows(gpu_ctx, rope, gpu_ctx.upload(x), False, 2 * dh, buf, False, 2 * dh, 0, dh, -1, 1, 1,
                   dh, pos, 70, used=gpu_ctx.upload(np.array([used], I32)))
        _, left = read()
        assert left[done:].all() and not left[:done].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dh,dtype", [(64, "bf16"), (64, "f32"), (48, "f32")])
def test_rope_rows_that_are_no_numbers(gpu_ctx, dh, dtype):
    """What is no number stays in its head, or without a norm in its pair; huge and tiny values."""
    from rembed_amd import tensor as T
    rng = np.random.default_rng(4)
    x = rng.standard_normal((6, 3, dh))
    x[1, 0, 5], x[2, 1, dh - 1], x[3, 2, 0] = np.nan, np.inf, -np.inf
    x[4], x[5] = x[4] * 1e15, x[5] * 1e-30
    img, val = F.typed(x.reshape(6, -1), dtype)
    pos = np.arange(10, 16).astype(I32)
    rope = T.Rope(gpu_ctx, dh)
    for norm in (None, T.Norm(None, 1e-6)):
        buf, read = marked(gpu_ctx, 6, 3 * dh, False)
        T.RopeRows(gpu_ctx, rope, gpu_ctx.upload(img), dtype == "bf16", 3 * dh, buf, False, 3 * dh, 0,
                   2 * dh, -1, 2, 1, dh, gpu_ctx.upload(pos), 6, norm, norm)
        got = read()[0].reshape(6, 3, dh)
        bad = np.zeros((6, 3, dh), bool)
        for r, h, d in ((1, 0, 5), (2, 1, dh - 1), (3, 2, 0)):
            bad[r, h, [d, (d + dh // 2) % dh] if norm is None else slice(None)] = True
        if norm is None:
            assert not np.isfinite(got[bad]).any()
        else:  # an infinite value makes its head 0 but where it stands
            assert np.isnan(got[1, 0]).all() and np.isnan(got[2, 1]).any() and np.isnan(got[3, 2]).any()
        clean = np.where(np.isfinite(val), val, 0).astype(np.float64).reshape(6, 3, dh)
        y, off = clean, np.zeros_like(clean)
        if norm is not None:
            y, off = R.head_norm(y, None, 1e-6)
        y, off = R.turn(y, off, pos, *R.frequencies(dh), True)
        assert (np.abs(got - y)[~bad] <= R.stored(y, off, False)[~bad]).all()


@pytest.mark.gpu
def test_rope_refusals(gpu_ctx):
    from rembed_amd import _lib as L
    from rembed_amd import tensor as T
    rope, buf = T.Rope(gpu_ctx, 64), gpu_ctx.alloc(1 << 20)
    far = At(buf, 1 << 19)
    ok = [gpu_ctx.h, rope.h, buf.ptr, 1, 512, far.ptr, 1, 512, 0, 256, -1, 4, 2, 64, buf.ptr, 5, None,
          None, None]

    def no(code, **kw):
        a = list(ok)
        for i, v in kw.items():
            a[int(i[1:])] = v
        F.refused(code, "rh_rope_rows", *a)

    no(L.RH_ERR_INVALID, a1=None)
    no(L.RH_ERR_SHAPE, a13=32)                       # rot of 64
    with T.Context(0) as other:
        no(L.RH_ERR_INVALID, a0=other.h)
    for i in (2, 5, 14):
        no(L.RH_ERR_INVALID, **{"a%d" % i: None})
    no(L.RH_ERR_SHAPE, a4=383)
    no(L.RH_ERR_SHAPE, a7=383)
    no(L.RH_ERR_SHAPE, a8=-1)
    no(L.RH_ERR_SHAPE, a9=255)                       # k on q's last column
    no(L.RH_ERR_SHAPE, a10=-2)
    no(L.RH_ERR_SHAPE, a10=128)
    no(L.RH_ERR_SHAPE, a10=385)                      # v behind the row
    no(L.RH_ERR_INVALID, a2=buf.ptr + 1)
    no(L.RH_ERR_INVALID, a14=buf.ptr + 2)
    no(L.RH_ERR_INVALID, a18=buf.ptr + 2)
    no(L.RH_ERR_INVALID, a5=buf.ptr + 2)             # out shifted on x
    no(L.RH_ERR_INVALID, a5=buf.ptr, a6=0)           # another type on x
    no(L.RH_ERR_INVALID, a5=buf.ptr, a7=520)
    for bad in (L.NormDesc(2, 0, None, None), L.NormDesc(1, -1, None, None),
                L.NormDesc(1, 0, 4098, None), L.NormDesc(1, 0, None, 4096)):
        no(L.RH_ERR_INVALID, a16=bad)
        no(L.RH_ERR_INVALID, a17=bad)
    assert L.lib.rh_rope_rows(*ok[:15], 0, *ok[16:]) == 0        # no rows
    assert L.lib.rh_rope_rows(*ok[:11], 0, 0, *ok[13:]) == 0     # no heads
    rope.close()
    odd = T.Rope(gpu_ctx, 24)
    cache = F.device_cache(gpu_ctx, O.Cache(2, 1, 64))
    args = [gpu_ctx.h, odd.h, cache.desc, buf.ptr, 1, 192, 0, 64, 128, far.ptr, 1, 64, 1, buf.ptr,
            buf.ptr, buf.ptr, buf.ptr, 1, 4, None, None]
    F.refused(L.RH_ERR_SHAPE, "rh_rope_append", *args)           # 24 is no multiple of 16
    good = T.Rope(gpu_ctx, 32)
    args[1] = good.h
    for i, v, code in ((0, None, L.RH_ERR_INVALID), (1, None, L.RH_ERR_INVALID),
                       (3, None, L.RH_ERR_INVALID), (9, None, L.RH_ERR_INVALID),
                       (13, None, L.RH_ERR_INVALID), (14, None, L.RH_ERR_INVALID),
                       (15, None, L.RH_ERR_INVALID), (16, None, L.RH_ERR_INVALID),
                       (5, 184, L.RH_ERR_SHAPE), (5, 196, L.RH_ERR_SHAPE), (6, 4, L.RH_ERR_SHAPE),
                       (7, -8, L.RH_ERR_SHAPE), (8, 136, L.RH_ERR_SHAPE), (11, 56, L.RH_ERR_SHAPE),
                       (3, buf.ptr + 8, L.RH_ERR_SHAPE), (9, far.ptr + 8, L.RH_ERR_SHAPE),
                       (13, buf.ptr + 2, L.RH_ERR_INVALID), (16, buf.ptr + 4, L.RH_ERR_INVALID),
                       (18, 2 ** 31 - 1, L.RH_ERR_SHAPE),
                       (9, buf.ptr + 16, L.RH_ERR_INVALID), (7, 0, L.RH_ERR_INVALID)):
        a = list(args)
        a[i] = v
        if i == 18:                                  # too many blocks, without q
            a[9], a[12] = None, 0
        if i == 7 and v == 0:                        # q on its columns of x, which are k's too
            a[9], a[11] = buf.ptr, 192
        F.refused(code, "rh_rope_append", *a)


# ---- GPU: residual norms ----------------------------------------------------------------

SIZES = [(1, 1), (3, 7), (5, 8), (4, 100), (2, 128), (130, 129), (7, 384), (1, 512), (300, 520),
         (3, 768), (9, 1000), (1030, 1024), (2, 1025), (5, 1544), (1, 2048), (3, 2049), (2, 2560),
         (6, 4096), (1, 5003), (2, 8192), (3, 8200), (1, 16384), (1, 16383), (1500, 640)]
KINDS = [("none", "none", "rms"), ("rms", "none", "rms"), ("layer", "row", "layer"),
         ("none", "channel", "layer"), ("rms", "row", "none"), (None, None, "rms"),
         (None, None, "layer"), ("layer", "channel", "rms"), ("none", "row", "none"),
         (None, None, "none")]
KIND = {"none": 0, None: 0, "rms": 1, "layer": 2}


def run_residual(ctx, x, y, res, m, n, xt, yt, sum_t, out_t, codes, pad=0, used=None):
    """x, y as device images; sum and out (float64), codes and scale bytes, and what is left."""
    from rembed_amd import tensor as T
    ld = n + pad
    total, rs = marked(ctx, m + 1, ld, xt == "bf16") if sum_t else (None, None)
    out, ro = marked(ctx, m + 1, ld, out_t == "bf16") if out_t else (None, None)
    ldq = T.ldq_fp8(n)
    qa = ctx.upload(np.full((m + 1, ldq), 0xAA, np.uint8)) if codes else None
    sa = ctx.upload(np.full(T.fp8_scale_bytes(m, n), 0xAA, np.uint8)) if codes else None
    T.ResidualNorm(ctx, res, x, xt == "bf16", ld, y, yt == "bf16", ld, total, ld, out,
                   out_t == "bf16", ld, qa, ldq if codes else 0, sa, m, n, used)
    got = {}
    for name, read in (("sum", rs), ("out", ro)):
        if read:
            v, left = read()
            assert left[m:].all() and left[:, n:].all()
            got[name] = v[:m, :n].astype(np.float64)
            got[name + "_left"] = left[:m, :n]
    if codes:
        ctx.sync()
        q = qa.download(np.uint8, (m + 1, ldq))
        assert (q[m:] == 0xAA).all()
        got["codes"] = q[:m]
        raw = sa.download(np.uint8, (T.fp8_scale_bytes(m, n),))
        got["scales"] = O.scale_rows(raw, m, ldq // 128)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("size", range(len(SIZES)), ids=lambda i: "%dx%d" % SIZES[i])
@pytest.mark.parametrize("turn", range(5))
def test_residual_norm(gpu_ctx, size, turn):
    from rembed_amd import tensor as T
    m, n = SIZES[size]
    case = size * 3 + turn * 7
    post, gate, pre = KINDS[(size + 2 * turn) % len(KINDS)]
    xt, yt = (("f32", "bf16"), ("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"))[case % 4]
    out_t = ("bf16", "f32", None)[case % 3]
    codes = out_t is None or case % 2 == 0
    pad = (0, 8, 3)[case % 3] if turn else 0
    rng = np.random.default_rng(case)
    xs, ys = ((1.0, 1.0), (0.5, 2.0), (1.0, -0.25))[case % 3]
    # columns of different sizes, rows around means of different sizes
    def data():
        v = rng.standard_normal((m, n + pad)) * np.exp(rng.uniform(-2, 2, n + pad))
        return v + rng.uniform(-3, 3, (m, 1))

    xi, xv = F.typed(data(), xt)
    yi, yv = F.typed(data(), yt)
    vec = lambda: rng.uniform(-1.5, 1.5, n).astype(np.float32)
    w = {k: vec() for k in ("post", "post_b", "pre", "pre_b")}
    d = {k: gpu_ctx.upload(v) for k, v in w.items()}
    eps = {"post": 1e-6, "pre": 1e-5}

    def norm(which, kind):
        if KIND[kind] == 0:
            return None, (0, None, None, 0)
        bias = kind == "layer" and case % 5 != 0
        weight = case % 7 != 0
        return (T.Norm(d[which] if weight else None, eps[which], d[which + "_b"] if bias else None,
                       layer=kind == "layer"),
                (KIND[kind], w[which].astype(np.float64) if weight else None,
                 w[which + "_b"].astype(np.float64) if bias else None, eps[which]))

    (n1, o1), (n2, o2) = norm("post", post), norm("pre", pre)
    g = ldg = None
    if gate in ("row", "channel"):
        ldg = n + 4 if gate == "row" else 0
        g = rng.uniform(-1, 2, (m, n + 4) if ldg else n).astype(np.float32)
    res = T.Residual(n1, n2, None if g is None else gpu_ctx.upload(g), ldg or 0, xs, ys)
    got = run_residual(gpu_ctx, gpu_ctx.upload(xi), gpu_ctx.upload(yi) if post else None, res, m, n, xt,
                       yt, turn != 3 or not (out_t or codes), out_t, codes, pad)
    gv = None if g is None else (g[:, :n] if ldg else g).astype(np.float64)
    s, so, want, far = R.residual(xv[:, :n].astype(np.float64), yv[:, :n].astype(np.float64)
                                  if post else None, o1, o2, gv, xs, ys)
    if "sum" in got:
        assert (np.abs(got["sum"] - s) <= R.stored(s, so, xt == "bf16")).all()
    if "out" in got:
        assert (np.abs(got["out"] - want) <= R.stored(want, far, out_t == "bf16")).all()
    if codes:
        check_codes(got, want, far, n)
        if out_t == "f32":  # the codes of the very values that are stored
            c, e, _ = O.quantize_rows(got["out"])
            assert np.array_equal(got["scales"], e)
            assert np.array_equal(O.CODES[got["codes"]], O.CODES[c])


def check_codes(got, want, far, n):
    """Codes times their scales within half a step of e4m3 of the values; scales that fit them."""
    assert (got["codes"][:, n:] == 0).all()
    scale = np.repeat(O.two(got["scales"].astype(np.int64)), 128, 1)[:, :n]
    v = O.CODES[got["codes"][:, :n]] * scale
    tol = far + 2.0 ** -4 * (np.abs(want) + far) + scale * 2.0 ** -10
    assert (np.abs(v - want) <= tol).all()
    for j in range(0, n, 128):
        b, f, e = np.abs(want[:, j:j + 128]), far[:, j:j + 128], got["scales"][:, j // 128].astype(int)
        lo, hi = O.exponent((b - f).max(1).clip(0)), O.exponent((b + f).max(1))
        assert ((e >= lo) & (e <= hi)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [768, 1001, 4096])
def test_residual_norm_in_place(gpu_ctx, n):
    """sum on x, out on y; out on x (a post-norm block); sum on y: the bits of other buffers'."""
    from rembed_amd import tensor as T
    rng = np.random.default_rng(n)
    m = 21
    xi, _ = F.typed(rng.standard_normal((m, n)), "bf16")
    yi, _ = F.typed(rng.standard_normal((m, n)), "bf16")
    w = gpu_ctx.upload(rng.uniform(0.5, 1.5, n).astype(np.float32))
    res = T.Residual(T.Norm(w), T.Norm(w, 1e-5, w, layer=True))

    def run(where_sum, where_out):
        x, y = gpu_ctx.upload(xi), gpu_ctx.upload(yi)
        bufs = {"x": x, "y": y, "z": gpu_ctx.alloc(xi.nbytes), "t": gpu_ctx.alloc(xi.nbytes)}
        T.ResidualNorm(gpu_ctx, res, x, True, n, y, True, n, bufs.get(where_sum), n,
                       bufs[where_out], True, n, None, 0, None, m, n)
        gpu_ctx.sync()
        return tuple(None if k is None else bufs[k].download(np.uint16, xi.shape)
                     for k in (where_sum, where_out))

    s, o = run("z", "t")
    for a, b in (("x", "y"), ("x", "t"), ("y", "x"), ("y", "t"), (None, "x"), (None, "y")):
        s2, o2 = run(a, b)
        assert np.array_equal(o, o2) and (s2 is None or np.array_equal(s, s2)), (a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [256, 1000, 1003, 4096])
def test_residual_norm_used(gpu_ctx, n):
    from rembed_amd import tensor as T
    m = 131
    x = np.ones((m, n), np.float32)
    res = T.Residual(None, T.Norm())
    for used, done in ((0, 0), (1, 1), (130, 130), (131, 131), (500, 131), (-1, 0)):
        got = run_residual(gpu_ctx, gpu_ctx.upload(x), None, res, m, n, "f32", "f32", True, "bf16", True,
                           used=gpu_ctx.upload(np.array([used], I32)))
        for name in ("sum", "out"):
            assert got[name + "_left"][done:].all() and not got[name + "_left"][:done].any()
        assert (got["codes"][done:] == 0xAA).all() and (got["codes"][:done, :n] != 0xAA).all()
        # values of 1 - 5e-7: 448 * 2^(119 - 127) = 1.75 holds them, 448 * 2^(118 - 127) does not
        assert (got["scales"][done:] == 0xAA).all() and (got["scales"][:done] == 119).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [512, 1003, 4096])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_residual_norm_of_odd_values(gpu_ctx, n, kind):
    """Rows of zeros, of one value, tiny and huge ones; what is no number stays in its row."""
    from rembed_amd import tensor as T
    rng = np.random.default_rng(n)
    x = rng.standard_normal((9, n))
    x[0], x[1] = 0.0, 3.0
    x[2] *= 1e-30
    x[3] *= 1e15
    x[4, n - 1], x[5, 0], x[6, 7] = np.nan, np.inf, -np.inf
    x[7] = 0.0
    x[7, 1] = 2.0 ** -140
    x[8] = 1000.0 + 0.01 * x[8]
    img, val = F.typed(x, "f32")
    res = T.Residual(None, T.Norm(None, 1e-6, None, layer=kind == "layer"))
    got = run_residual(gpu_ctx, gpu_ctx.upload(img), None, res, 9, n, "f32", "f32", True, "f32", True)
    assert np.array_equal(got["sum"], val.astype(np.float64), equal_nan=True)
    fine = [0, 1, 2, 3, 7, 8]
    _, _, want, far = R.residual(val[fine].astype(np.float64), None, (0, None, None, 0),
                                 (KIND[kind], None, None, 1e-6), None, 1.0, 1.0)
    assert (np.abs(got["out"][fine] - want) <= R.stored(want, far, False)).all()
    for r, at_ in ((4, slice(None)), (5, 0), (6, 7)):
        assert np.isnan(got["out"][r, at_]).all()
        assert np.isnan(O.CODES[got["codes"][r, :n]][at_]).all()
    c, e, _ = O.quantize_rows(got["out"])
    assert np.array_equal(got["scales"], e)
    assert np.array_equal(O.CODES[got["codes"]], O.CODES[c], equal_nan=True)


# ---- GPU: the rotary append, the cache read back -------------------------------------------

APPEND = [  # heads, kv, dh, rot, layout, lengths of three steps
    (16, 8, 128, 128, 0, ([1], [1], [63])), (3, 1, 256, 64, 1, ([65, 3], [1, 0], [2, 130])),
    (2, 2, 64, 64, 0, ([0, 64, 5], [200, 1, 1], [1, 1, 1])), (4, 2, 64, 32, 0, ([31, 33], [1, 1], [90, 2])),
    (0, 3, 128, 32, 1, ([10, 20], [60, 1], [1, 1])), (8, 1, 128, 16, 0, ([1, 1, 1, 1], [2, 3, 4, 5], [70, 0, 0, 1])),
    (3, 3, 256, 256, 0, ([100], [28], [1])), (6, 2, 64, 16, 1, ([7] * 70, [1] * 70, [60] * 70)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("i", range(len(APPEND)), ids=lambda i: "%dx%d-%d-%d-%d" % APPEND[i][:5])
@pytest.mark.parametrize("normed", [False, True])
def test_rope_append(gpu_ctx, i, dtype, normed):
    """Three steps into one cache: q's rows, and the cache's bytes as rh_cache_append's of the
    rows that rh_rope_rows gives in fp32 (with a norm, whose sums are added in another order,
    within a step of e4m3 of the values)."""
    from rembed_amd import tensor as T
    heads, kv, dh, rot, layout, steps = APPEND[i]
    rng = np.random.default_rng(i)
    n = len(steps[0])
    total = [sum(s[b] for s in steps) for b in range(n)]
    pages, table, _, _, _, _ = F.batch_of(rng, [0] * n, total)
    c = O.Cache(pages, kv, dh)
    dev = F.device_cache(gpu_ctx, c)
    rope = T.Rope(gpu_ctx, rot, theta=1e4, layout=layout, scaling=3, factor=2.0, original=512)
    w = [rng.uniform(0.5, 1.5, dh).astype(np.float32) for _ in "qk"]
    norms = [T.Norm(gpu_ctx.upload(a), 1e-6) for a in w] if normed else [None, None]
    past = [0] * n
    bf, front = dtype == "bf16", 8 * (i % 3)
    width = (heads + 2 * kv) * dh + front
    for step, fresh in enumerate(steps):
        rows = sum(fresh)
        cu, blk, lens, slots, pos, _ = O.plan(past, fresh, [
            table[b, j] for b in range(n)
            for j in range(-(-past[b] // 64), -(-(past[b] + fresh[b]) // 64))], table.copy(), rows + 3)
        x = rng.standard_normal((rows + 3, width)) * np.exp(rng.uniform(-2, 2, (rows + 3, 1)))
        img, val = F.typed(x, dtype)
        d, dpos = gpu_ctx.upload(img), gpu_ctx.upload(pos)
        off = (front, front + heads * dh, front + (heads + kv) * dh)
        turned, read_turned = marked(gpu_ctx, rows + 3, width, False)
        T.RopeRows(gpu_ctx, rope, d, bf, width, turned, False, width, off[0], off[1], off[2], heads,
                   kv, dh, dpos, rows, *norms)
        turned, _ = read_turned()
        k = turned[:rows, off[1]:off[2]].reshape(rows, kv, dh).astype(np.float64)
        v = turned[:rows, off[2]:].reshape(rows, kv, dh).astype(np.float64)
        q_bf = (i + step) % 2 == 0
        q, read_q = marked(gpu_ctx, rows + 3, heads * dh + 8, q_bf)
        T.RopeAppend(gpu_ctx, rope, dev, d, bf, width, *off, q if heads else None, q_bf,
                     heads * dh + 8, heads, dpos, gpu_ctx.upload(cu), gpu_ctx.upload(blk),
                     gpu_ctx.upload(slots), n, rows + 3, *norms)
        got, left = read_q()
        assert left[rows:].all() and left[:, heads * dh:].all()
        if heads:
            val = val[:rows, front:].astype(np.float64).reshape(rows, -1, dh)
            check_heads(got[:rows, :heads * dh].reshape(rows, heads, dh), val[:, :heads], heads, 0, dh,
                        rot, layout, dict(theta=1e4, scaling=3, factor=2.0, original=512), pos[:rows],
                        w if normed else None, q_bf)
        before = [a.copy() for a in (c.k, c.k_exp)]
        c.append(k, v, cu, slots)
        if normed:
            same_but_for_norms(dev, c, before)
        else:
            F.same_cache(dev, c)
        past = [p + f for p, f in zip(past, fresh)]


def same_but_for_norms(dev, c, before):
    """K's values where two norms may differ by 36 u: codes a step apart, where the value lies
    between them; V equal. c then holds what the device does."""
    k = dev.k.download(np.uint8, c.k.shape)
    e = dev.k_exp.download(np.uint8, c.k_exp.shape)
    assert np.array_equal(dev.v.download(np.uint8, c.v.shape) & 127 != 0, c.v & 127 != 0)
    assert np.array_equal(O.CODES[dev.v.download(np.uint8, c.v.shape)], O.CODES[c.v], equal_nan=True)
    assert np.array_equal(dev.v_exp.download(np.uint8, c.v_exp.shape), c.v_exp)
    old = O.CODES[c.k] * O.two(c.k_exp.astype(np.int64))[:, :, None]
    new = O.CODES[k] * O.two(e.astype(np.int64))[:, :, None]
    differ = ~((old == new) | (np.isnan(old) & np.isnan(new)))
    scale = O.two(np.maximum(e, c.k_exp).astype(np.int64))[:, :, None]
    assert (np.abs(old - new)[differ] <= (2.0 ** -3 * np.maximum(np.abs(old), np.abs(new)) * (1 + 2.0 ** -3)
                                          + scale * 2.0 ** -9)[differ]).all()
    # values that lie within 36 u of a border between two codes are rare
    assert differ.mean() <= 1e-3 and (e != c.k_exp).mean() <= 0.05
    c.k, c.k_exp = k, e


@pytest.mark.gpu
def test_rope_append_on_its_own_rows(gpu_ctx):
    """q in place: the bits of another buffer's, k's and v's columns left."""
    from rembed_amd import tensor as T
    rng = np.random.default_rng(8)
    heads, kv, dh, n = 4, 2, 64, 90
    width = (heads + 2 * kv) * dh + 8
    img, _ = F.typed(rng.standard_normal((n, width)), "bf16")
    cu, blk, lens, slots, pos, _ = O.plan([0], [n], [1, 0], np.zeros((1, 2), I32), n)
    rope, norm = T.Rope(gpu_ctx, 64), T.Norm(None, 1e-6)
    got = []
    for place in (False, True):
        dev = F.device_cache(gpu_ctx, O.Cache(2, kv, dh))
        x = gpu_ctx.upload(img)
        q = At(x, 16) if place else gpu_ctx.alloc(n * width * 2)
        T.RopeAppend(gpu_ctx, rope, dev, x, True, width, 8, 8 + heads * dh, 8 + (heads + kv) * dh, q, True,
                     width, heads, gpu_ctx.upload(pos), gpu_ctx.upload(cu), gpu_ctx.upload(blk),
                     gpu_ctx.upload(slots), 1, n, norm, norm)
        gpu_ctx.sync()
        rows = (x if place else q).download(np.uint16, (n, width))
        got.append((rows[:, 8:8 + heads * dh] if place else rows[:, :heads * dh],
                    [getattr(dev, a).download(np.uint8, (getattr(dev, a).nbytes,))
                     for a in ("k", "v", "k_exp", "v_exp")]))
        if place:
            assert np.array_equal(rows[:, :8], img[:, :8])
            assert np.array_equal(rows[:, 8 + heads * dh:], img[:, 8 + heads * dh:])
    assert np.array_equal(got[0][0], got[1][0])
    for a, b in zip(got[0][1], got[1][1]):
        assert np.array_equal(a, b)


@pytest.mark.gpu
def test_rope_append_of_what_has_no_page_or_is_no_number(gpu_ctx):
    from rembed_amd import tensor as T
    rng = np.random.default_rng(9)
    heads, kv, dh = 1, 2, 64
    width = (heads + 2 * kv) * dh
    x = rng.standard_normal((12, width)).astype(np.float32)
    x[5, 64 + 3] = np.nan          # K of head 0
    x[6, 64 + 128 + 64] = np.inf   # V of head 1
    slots = np.array([-1, -1, 128, 129, 130, 64, 65, 66, -1, -1, -1, -1], np.int64)
    cu, blk = np.array([0, 2, 5, 8], I32), np.array([0, 1, 2, 3], I32)
    pos = np.zeros(12, I32)
    c = O.Cache(2, kv, dh)
    dev = F.device_cache(gpu_ctx, c)
    rope = T.Rope(gpu_ctx, 64)

    def go(cache, cu, blk, slots):
        q, read = marked(gpu_ctx, 12, 64, False)
        T.RopeAppend(gpu_ctx, rope, cache, gpu_ctx.upload(x), False, width, 0, 64, 64 + 128, q, False, 64,
                     heads, gpu_ctx.upload(pos), gpu_ctx.upload(cu), gpu_ctx.upload(blk),
                     gpu_ctx.upload(slots), 3, 12)
        return read()

    got, left = go(dev, cu, blk, slots)
    assert np.array_equal(got[:8], x[:8, :64]) and left[8:].all()
    c.append(x[:, 64:192].reshape(12, 2, 64).astype(np.float64),
             x[:, 192:].reshape(12, 2, 64).astype(np.float64), cu, slots)
    F.same_cache(dev, c)
    zero = np.zeros(4, I32)
    got, left = go(dev, zero, zero, np.full(12, -1, np.int64))  # a plan that failed
    assert left.all()
    F.same_cache(dev, c)
    none = T.KVCache(gpu_ctx, 0, kv, dh)                        # a cache of no pages: q alone
    got, left = go(none, cu, blk, slots)
    assert np.array_equal(got[:8], x[:8, :64]) and left[8:].all()


@pytest.mark.gpu
@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 70])
def test_rope_append_of_zeros_and_extremes(gpu_ctx, dh, n):
    """Heads of zeros (whose 1 / rms is 1 / sqrt(eps)), tiny and huge ones, alone in their blocks and
    together: the codes of the rows that rh_rope_rows gives."""
    from rembed_amd import tensor as T
    rng = np.random.default_rng(dh + n)
    rope, norm = T.Rope(gpu_ctx, dh), T.Norm(None, 1e-6)
    for scale in (0.0, 1e-30, 2.0 ** -140, 1e15, None):
        x = rng.standard_normal((n, 2 * dh))
        x[:, :dh] *= np.exp(rng.uniform(-60, 30, (n, 1))) if scale is None else scale
        img, val = F.typed(x, "f32")
        c = O.Cache(2, 1, dh)
        dev = F.device_cache(gpu_ctx, c)
        cu, blk, lens, slots, pos, _ = O.plan([0], [n], [1, 0], np.zeros((1, 2), I32), n)
        d, dpos = gpu_ctx.upload(img), gpu_ctx.upload(pos)
        turned, read = marked(gpu_ctx, n, 2 * dh, False)
        T.RopeRows(gpu_ctx, rope, d, False, 2 * dh, turned, False, 2 * dh, 0, 0, -1, 0, 1, dh, dpos, n, None,
                   norm)
        T.RopeAppend(gpu_ctx, rope, dev, d, False, 2 * dh, 0, 0, dh, None, False, 0, 0, dpos,
                     gpu_ctx.upload(cu), gpu_ctx.upload(blk), gpu_ctx.upload(slots), 1, n, None, norm)
        k = read()[0][:, :dh].reshape(n, 1, dh).astype(np.float64)
        assert np.isfinite(k).all() and (scale != 0.0 or not k.any())
        c.append(k, val[:, dh:].reshape(n, 1, dh).astype(np.float64), cu, slots)
        same_but_for_norms(dev, c, None)


def filled(rng, ctx, pages, kv, dh):
    """A cache of random codes (NaN among them) and scales."""
    c = O.Cache(pages, kv, dh)
    c.k = rng.integers(0, 256, c.k.shape).astype(np.uint8)
    c.v = rng.integers(0, 256, c.v.shape).astype(np.uint8)
    c.k_exp = rng.integers(100, 150, c.k_exp.shape).astype(np.uint8)
    c.v_exp = rng.integers(0, 150, c.v_exp.shape).astype(np.uint8)
    return c, F.device_cache(ctx, c)


READ = [  # first positions, counts
    ([0], [1]), ([0], [64]), ([5], [200]), ([63, 64, 0], [1, 1, 65]), ([10, 0, 100], [0, 130, 0]),
    ([0, 37, 64, 1], [3, 300, 64, 63]), ([2] * 70, [5] * 70), ([1], [1000]), ([127, 0], [2, 0]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("i", range(len(READ)))
def test_cache_read(gpu_ctx, dh, out, i):
    from rembed_amd import tensor as T
    first, count = READ[i]
    rng = np.random.default_rng(i)
    kv, n = 1 + i % 3, len(first)
    pages, table, _, _, _, _ = F.batch_of(rng, [0] * n, [a + b for a, b in zip(first, count)])
    c, dev = filled(rng, gpu_ctx, pages, kv, dh)
    cu = np.concatenate([[0], np.cumsum(count)]).astype(I32)
    rows, width = int(cu[-1]), kv * dh
    ld = 2 * width + 24
    buf, read = marked(gpu_ctx, rows + 3, ld, out == "bf16")
    T.CacheRead(gpu_ctx, dev, gpu_ctx.upload(table), table.shape[1], gpu_ctx.upload(cu),
                None if not any(first) else gpu_ctx.upload(np.array(first, I32)), n, rows + 3, buf,
                out == "bf16", ld, width + 16, 8)  # V before K
    got, left = read()
    assert left[rows:].all() and left[:, :8].all() and left[:, 8 + width:16 + width].all()
    assert left[:, 16 + 2 * width:].all()
    for b in range(n):
        k, v = c.rows(table[b], first[b] + count[b])
        for want, col in ((k, width + 16), (v, 8)):
            w = want[first[b]:].reshape(count[b], width)
            g = got[cu[b]:cu[b + 1], col:col + width]
            if out == "bf16":
                w = F.bf16(w)[0]
            assert np.array_equal(g, w.astype(np.float32), equal_nan=True)


@pytest.mark.gpu
def test_cache_read_of_what_is_not_there(gpu_ctx):
    """Pages that are none, positions before 0 and behind the table, row offsets that go down."""
    from rembed_amd import tensor as T
    rng = np.random.default_rng(3)
    c, dev = filled(rng, gpu_ctx, 4, 1, 64)
    c.k_exp[:], c.v_exp[:] = 127, 127
    dev = F.device_cache(gpu_ctx, c)
    table = np.array([[2, -1, 1], [0, 4, 2 ** 31 - 1], [3, 3, 3], [1, 2, 0]], I32)
    first = np.array([0, 30, -70, 128], I32)
    count = [192, 100, 80, 100]
    cu = np.concatenate([[0], np.cumsum(count)]).astype(I32)
    rows = int(cu[-1])
    buf, read = marked(gpu_ctx, rows, 128, False)
    T.CacheRead(gpu_ctx, dev, gpu_ctx.upload(table), 3, gpu_ctx.upload(cu), gpu_ctx.upload(first), 4,
                rows, buf, False, 128, 0, 64)
    got, left = read()
    for b in range(4):
        for t in range(count[b]):
            p = int(first[b]) + t
            page = table[b, p // 64] if 0 <= p < 192 else -1
            k, v = c.rows([page], 64) if 0 <= page < 4 else (np.zeros((64, 1, 64)),) * 2
            row = got[cu[b] + t]
            assert np.array_equal(row[:64], k[p % 64, 0].astype(np.float32), equal_nan=True)
            assert np.array_equal(row[64:], v[p % 64, 0].astype(np.float32), equal_nan=True)
    for bad in ([0, -5, 10, 10, 10], [-3, 5, 5, 5, 5], [0, 0, 0, 0, rows + 1], [9, 4, 4, 4, 4]):
        buf, read = marked(gpu_ctx, rows, 128, False)
        bad = np.array(bad, I32)
        T.CacheRead(gpu_ctx, dev, gpu_ctx.upload(table), 3, gpu_ctx.upload(bad), None, 4, rows, buf,
                    False, 128, 0, 64)
        _, left = read()
        assert left[max(0, int(bad.max())):].all()
