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
import test_row_operators as W

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


# ---- outputs on what a call reads -------------------------------------------------------------

def test_residual_overlaps():
    """An output that holds the weights, the gate, the count or the scales is refused to the byte;
    what lies between an output's rows, or next to them, is not."""
    from rembed_amd import _lib as L
    out, codes, scales = 4 << 20, 5 << 20, 6 << 20   # 9 rows of 256 values, 512 apart; codes; 2 * 128 bytes
    n, m, ld = 256, 9, 512
    end = out + 8 * ld * 4 + n * 4

    def call(post=L.NormDesc(), pre=L.NormDesc(), gate=None, ldg=0, used=None, sa=scales):
        return ["rh_residual_norm", L.ResidualDesc(post, pre, gate, ldg, 1.0, 1.0), at(1 << 20), 0, n,
                at(2 << 20), 0, n, None, 0, at(out), 0, ld, at(codes), n, at(sa), m, n, used]

    def no(**kw):
        fn, *args = call(**kw)
        F.refused(L.RH_ERR_INVALID, fn, None, *args)
        assert b"overlaps" in L.lib.rh_last_error()

    gaps = [out + i * ld * 4 + n * 4 for i in range(m)]
    for p in gaps + [out - n * 4, end, codes - n * 4, codes + m * n, scales - n * 4, scales + 256]:
        for norm in (L.NormDesc(1, 0, p, None), L.NormDesc(2, 0, None, p)):
            passes(*call(pre=norm))
            passes(*call(post=norm))
        passes(*call(used=at(p)))
    for p in [out, end - 4, codes, codes + m * n - 4, scales, scales + 252] + [g - 4 for g in gaps]:
        for norm in (L.NormDesc(1, 0, p, None), L.NormDesc(2, 0, None, p), L.NormDesc(1, 0, p - n * 4 + 4, None)):
            no(pre=norm)
            no(post=norm)
        no(used=at(p))
    no(pre=L.NormDesc(1, 0, gaps[0] + 4, None))      # on the next row's first value
    no(gate=out + 4 * ld, ldg=ld)
    no(gate=scales + 252)
    for p in gaps:
        passes(*call(sa=p))
    for p in (out, gaps[3] - 4, end - 4, codes + 4, 1 << 20, (2 << 20) + m * n * 4 - 4):
        no(sa=p)


def test_read_overlaps():
    """Rows of K and V on the cache, the table, the offsets or the first positions."""
    from rembed_amd import _lib as L
    k, v, ke, ve, table, cu, first, out = (i << 20 for i in range(1, 9))
    codes, rows, batch, ldt = 4 * 2 * 64 * 64, 9, 2, 4   # 4 pages of 2 heads of 64; rows of 8 + 2 * 128, 300 apart

    def call(**kw):
        p = dict(k=k, v=v, ke=ke, ve=ve, table=table, cu=cu, first=first)
        p.update(kw)
        return ["rh_cache_read", F.desc(4, 2, 64, p["k"], p["v"], p["ke"], p["ve"]), at(p["table"]), ldt,
                at(p["cu"]), at(p["first"]), batch, rows, at(out), 0, 304, 8, 136]

    sizes = dict(k=codes, v=codes, ke=8, ve=8, table=batch * ldt * 4, cu=12, first=8)
    end = out + (8 * 304 + 264) * 4
    for name, size in sizes.items():
        # in front of the first row's columns, behind the last's, between two rows where it fits
        near = [out + 32 - (size + 15) // 16 * 16, end] + [out + (i * 304 + 264) * 4 for i in range(8) if size <= 160]
        for p in near:
            passes(*call(**{name: p}))
        for p in (out + 32, end - 16, out + (3 * 304 + 260) * 4, out + (4 * 304 + 136) * 4):
            fn, *args = call(**{name: p})
            F.refused(L.RH_ERR_INVALID, fn, None, *args)
            assert b"overlaps" in L.lib.rh_last_error(), name


@pytest.mark.gpu
def test_rotary_overlaps(gpu_ctx):
    """Rotary rows and the rotary append: outputs on weights, positions, tables, the cache. Every
    refusal is the host's."""
    from rembed_amd import _lib as L
    from rembed_amd import tensor as T
    rope, buf = T.Rope(gpu_ctx, 32), gpu_ctx.upload(np.zeros(1 << 23, np.uint8))
    x, out, pos, used, w = (buf.ptr + (i << 20) for i in range(5))
    rms = lambda p: L.NormDesc(1, 0, p, None)

    def rows(pos=pos, used=used, q=rms(w), k=rms(w + 256)):
        return [gpu_ctx.h, rope.h, x, 1, 528, out, 0, 528, 8, 264, 392, 4, 2, 64, pos, 9, q, k, used]

    last = out + (8 * 528 + 392 + 128) * 4               # behind v's last value
    inside = [out + 32, out + 264 * 4, last - 4, out + (528 + 8) * 4]
    for p in inside:
        for kw in (dict(pos=p), dict(used=p), dict(q=rms(p)), dict(k=rms(p)), dict(pos=p - 32), dict(k=rms(p - 252))):
            F.refused(L.RH_ERR_INVALID, "rh_rope_rows", *rows(**kw))
            assert b"overlaps" in L.lib.rh_last_error()

    k, v, ke, ve, cu, blk, slots = (buf.ptr + (5 << 20) + (i << 17) for i in range(7))
    codes = 2 * 64 * 64                                  # two pages of one head

    def app(k=k, v=v, ke=ke, ve=ve, cu=cu, blk=blk, slots=slots, pos=pos, qn=rms(w), kn=rms(w + 256)):
        return [gpu_ctx.h, rope.h, F.desc(2, 1, 64, k, v, ke, ve), x, 1, 512, 8, 264, 392, out, 1, 512, 4, pos,
                cu, blk, slots, 2, 9, qn, kn]

    q_end = out + (8 * 512 + 256) * 2
    for name in ("k", "v", "ke", "ve", "cu", "blk", "slots", "pos", "qn", "kn"):
        take = rms if name in ("qn", "kn") else int
        on_q = [out, out + 16, q_end - 16, out + 512 * 2 * 3 + 496]
        on_x = [x, x + (8 * 512 + 448) * 2] if name in ("k", "v", "ke", "ve") else []
        on_cache = [] if name in ("k", "v", "ke", "ve") else [k, v + codes - 8, ke, ve]
        for p in on_q + on_x + on_cache:
            F.refused(L.RH_ERR_INVALID, "rh_rope_append", *app(**{name: take(p)}))
            assert b"overlaps" in L.lib.rh_last_error(), (name, p)


@pytest.mark.gpu
def test_rotary_rows_beside_what_they_read(gpu_ctx):
    """Weights, positions and the count between the output's rows: the bits of other places."""
    from rembed_amd import tensor as T
    rng = np.random.default_rng(5)
    rope, n, dh = T.Rope(gpu_ctx, 64), 7, 64
    ld = 2 * dh + 96                                     # 96 values between two rows
    img = rng.standard_normal((n, 2 * dh)).astype(np.float32)
    x = gpu_ctx.upload(img)
    pos, w = rng.integers(0, 999, n).astype(I32), rng.uniform(0.5, 1.5, dh).astype(np.float32)

    class At:
        def __init__(self, buf, value):
            self.ptr = buf.ptr + 4 * value

    got = []
    for inside in (False, True):
        host = np.zeros((n, ld), np.float32)
        host[0, 2 * dh:2 * dh + n] = pos.view(np.float32)
        host[1, 2 * dh + 32:] = w
        host[2, 2 * dh + 5] = np.array([n - 1], I32).view(np.float32)[0]
        buf = gpu_ctx.upload(host)
        place = buf if inside else gpu_ctx.upload(host)
        norm = T.Norm(At(place, ld + 2 * dh + 32), 1e-6)
        T.RopeRows(gpu_ctx, rope, x, False, 2 * dh, buf, False, ld, 0, dh, -1, 1, 1, dh, At(place, 2 * dh), n,
                   norm, norm, At(place, 2 * ld + 2 * dh + 5))
        gpu_ctx.sync()
        got.append(buf.download(np.uint32, (n, ld)))
        assert np.array_equal(got[-1][:, 2 * dh:], host.view(np.uint32)[:, 2 * dh:])
        assert not got[-1][n - 1, :2 * dh].any()
    assert np.array_equal(*got) and got[0][:n - 1, :2 * dh].any(1).all()


def test_misaligned_tables_of_a_read():
    from rembed_amd import _lib as L
    ok = [None, F.desc(), F.P, 4, F.P, None, 2, 9, at(1 << 20), 1, 256, 0, 128]
    for i in (2, 4, 5):
        a = list(ok)
        a[i] = at(4098)
        F.refused(L.RH_ERR_INVALID, "rh_cache_read", *a)
        assert b"misaligned" in L.lib.rh_last_error()


@pytest.mark.gpu
def test_misaligned_tables_of_a_rotary_append(gpu_ctx):
    from rembed_amd import _lib as L
    from rembed_amd import tensor as T
    rope, buf = T.Rope(gpu_ctx, 32), gpu_ctx.upload(np.zeros(1 << 20, np.uint8))
    p = [buf.ptr + (i << 16) for i in range(10)]
    ok = [gpu_ctx.h, rope.h, F.desc(2, 1, 64, p[0], p[1], p[2], p[3]), p[4], 1, 192, 0, 64, 128, p[5], 1, 64, 1,
          p[6], p[7], p[8], p[9], 1, 4, None, None]
    for i in (14, 15):
        a = list(ok)
        a[i] += 2
        F.refused(L.RH_ERR_INVALID, "rh_rope_append", *a)
        assert b"misaligned" in L.lib.rh_last_error()
    assert L.lib.rh_rope_append(*ok) == 0                # of no rows: every offset is 0
    gpu_ctx.sync()


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


def test_rope_amp_that_fp32_does_not_hold():
    from rembed_amd import _lib as L
    from rembed_amd import tensor as T
    big = float(np.finfo(np.float32).max)
    assert T.rope_frequencies(8, amp=big)[1] == big
    for amp in (2.0 ** 128, 1e300):
        with pytest.raises(L.RembedError):
            T.rope_frequencies(8, amp=amp)


@pytest.mark.gpu
def test_rope_of_given_frequencies_of_any_size(gpu_ctx):
    """Angles within 2^-31 of a turn at every position: a sine near a whole turn shows them. Sine and
    cosine are those of pi from whole numbers."""
    from rembed_amd import tensor as T
    rng = np.random.default_rng(0)
    pi = machin()
    assert abs(pi / (1 << BITS) - np.pi) < 1e-15
    freq = [0.0, 5e-324, 1e-30, 2.0 ** -40, 0.37, 1.0, np.pi, 2 * np.pi, 50.0, -50.0, 1e3, -12345.678, 1e6,
            2.0 ** 53, 1e16, -3e18, 2.0 ** 63, 2.0 ** 64, 1e20, -1e25, 1e30, 1.7e38, 2.0 ** 127, 1e50, -1e77,
            1e100, 1e150, 2.0 ** 640, 1e200, -1e250, 1e300, np.finfo(np.float64).max]
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


# ---- GPU: many heads at document sizes -----------------------------------------------------

# rows, heads, kv, dh, rot, layout, dtype, out, in place, normed. Four heads a thread from heads * threads a head
# * rows = 2^19 on (value by value: from 8192 heads), the heads no multiple of four in most.
MANY = [
    (3000, 16, 8, 128, 128, 0, "bf16", "bf16", False, True), (5100, 5, 4, 128, 64, 1, "bf16", "f32", False, True),
    (2100, 9, 4, 128, 128, 0, "f32", "bf16", False, False), (2600, 9, 4, 128, 32, 0, "f32", "f32", True, True),
    (9500, 9, 5, 64, 64, 1, "bf16", "bf16", True, True), (3300, 11, 5, 64, 32, 0, "f32", "f32", False, True),
    (9100, 17, 6, 32, 32, 0, "bf16", "bf16", False, False), (5600, 4, 1, 256, 128, 0, "bf16", "bf16", False, True),
    (2800, 3, 2, 256, 256, 1, "f32", "bf16", False, True),
    # odd heads: runs of 8, 4 and 2 values, and value by value
    (9400, 5, 2, 80, 80, 0, "bf16", "bf16", True, True), (3400, 5, 4, 72, 72, 0, "bf16", "f32", False, False),
    (2100, 5, 2, 96, 50, 1, "bf16", "bf16", False, True), (2400, 5, 2, 36, 20, 0, "f32", "f32", True, True),
    (1100, 5, 2, 36, 18, 0, "bf16", "bf16", False, True), (1200, 6, 1, 254, 250, 0, "f32", "bf16", False, True),
    (1250, 5, 2, 254, 250, 0, "bf16", "bf16", True, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(len(MANY)), ids=lambda i: "%dx%d+%d-%d-%d-%d-%s-%s" % MANY[i][:8])
def test_rope_rows_of_many_heads(gpu_ctx, i):
    """Every q and k head of every row against 64 bits, v's copied (in place: left), what lies around
    the heads left as it was."""
    from rembed_amd import tensor as T
    rows, heads, kv, dh, rot, layout, dtype, out, place, normed = MANY[i]
    rng = np.random.default_rng(100 + i)
    front, nh = 8, heads + 2 * kv
    ld = front + nh * dh + 8
    x = rng.standard_normal((rows, ld)) * np.exp(rng.uniform(-3, 3, (rows, 1)))
    img, val = F.typed(x, dtype)
    pos = rng.integers(0, 200000, rows).astype(I32)
    w = [rng.uniform(0.5, 1.5, dh).astype(np.float32) for _ in "qk"]
    norms = [T.Norm(gpu_ctx.upload(a), e) for a, e in zip(w, (1e-6, 1e-3))] if normed else [None, None]
    rope = T.Rope(gpu_ctx, rot, layout=layout)
    src = gpu_ctx.upload(img)
    if place:
        buf, read = src, lambda: (gpu_ctx.sync(), src.download(img.dtype, (rows, ld)))[1]
    else:
        buf, read = W.marked(gpu_ctx, rows + 1, ld, out == "bf16")
    at_ = (front, front + heads * dh, front + (heads + kv) * dh)
    T.RopeRows(gpu_ctx, rope, src, dtype == "bf16", ld, buf, out == "bf16", ld, *at_, heads, kv, dh,
               gpu_ctx.upload(pos), rows, *norms)
    if place:
        bits = read()
        got = F.from_bf16(bits) if dtype == "bf16" else bits
        same = bits == img
        assert same[:, :front].all() and same[:, at_[2]:].all()
    else:
        got, left = read()
        assert left[rows:].all() and left[:, :front].all() and left[:, front + nh * dh:].all()
        got = got[:rows]
        v = val[:, at_[2]:front + nh * dh]
        v = F.bf16(v)[0] if out == "bf16" else v
        assert np.array_equal(got[:, at_[2]:front + nh * dh], v)
    heads_of = lambda a: a[:, front:at_[2]].astype(np.float64).reshape(rows, heads + kv, dh)
    W.check_heads(heads_of(got), heads_of(val), heads, kv, dh, rot, layout, {}, pos, w if normed else None,
                  out == "bf16")


# batch, lengths up to, cached before up to, heads, kv, dh, rot, layout, dtype, q in place. Threads of a
# token of heads of 128: eight up to 512 blocks, then four; heads of a thread's q: four from
# heads * threads a head * rows = 2^19 on.
APPENDS = [
    (40, 12, 130, 16, 8, 128, 128, 0, "bf16", False),      # four threads a token, one head a thread
    (7, 800, 90, 18, 8, 128, 128, 0, "bf16", False),       # four and four
    (19, 160, 70, 17, 8, 128, 64, 1, "f32", False),
    (9, 700, 100, 16, 8, 128, 128, 1, "bf16", True),
    (4, 2100, 50, 11, 1, 128, 128, 0, "bf16", False),      # eight and four
    (3, 3300, 70, 19, 2, 64, 64, 0, "bf16", False), (5, 1100, 0, 17, 3, 64, 32, 1, "f32", False),
    (3, 2300, 40, 7, 1, 256, 256, 0, "bf16", False), (3, 1200, 300, 6, 2, 256, 64, 1, "f32", False),
]


def append_case(ctx, i, normed):
    """A step behind cached beginnings: K and V as numbers, the cache before and after, q's rows."""
    from rembed_amd import tensor as T
    batch, most, before, heads, kv, dh, rot, layout, dtype, place = APPENDS[i]
    rng = np.random.default_rng(200 + i)
    fresh = rng.integers(most // 2 + 1, most + 1, batch)
    fresh[0] = most
    past = rng.integers(0, before + 1, batch)
    rows = int(fresh.sum())
    pages, table, _, _, _, _ = F.batch_of(rng, [0] * batch, past + fresh)
    free = [int(table[b, j]) for b in range(batch)
            for j in range(-(-past[b] // 64), -(-(past[b] + fresh[b]) // 64))]
    cu, blk, _, slots, pos, _ = O.plan(past, fresh, free, table.copy(), rows + 2)
    c = O.Cache(pages, kv, dh)
    c.k, c.v = (rng.integers(0, 127, a.shape).astype(np.uint8) | rng.integers(0, 2, a.shape).astype(np.uint8) << 7
                for a in (c.k, c.v))
    c.k_exp, c.v_exp = (rng.integers(112, 124, a.shape).astype(np.uint8) for a in (c.k_exp, c.v_exp))
    dev = F.device_cache(ctx, c)
    width = (heads + 2 * kv) * dh + 8
    x = rng.standard_normal((rows + 2, width)) * np.exp(rng.uniform(-2, 2, (rows + 2, 1)))
    img, val = F.typed(x, dtype)
    w = [rng.uniform(0.5, 1.5, dh).astype(np.float32) for _ in "qk"]
    norms = [T.Norm(ctx.upload(a), e) for a, e in zip(w, (1e-6, 1e-3))] if normed else [None, None]
    rope, src, bf = T.Rope(ctx, rot, layout=layout), ctx.upload(img), dtype == "bf16"
    if place:
        q, ldq, q_bf = W.At(src, 8 * img.itemsize), width, bf
    else:
        ldq, q_bf = heads * dh + 8, True
        q, read = W.marked(ctx, rows + 2, ldq, True)
    T.RopeAppend(ctx, rope, dev, src, bf, width, 8, 8 + heads * dh, 8 + (heads + kv) * dh, q, q_bf, ldq, heads,
                 ctx.upload(pos), ctx.upload(cu), ctx.upload(blk), ctx.upload(slots), batch, rows + 2, *norms)
    ctx.sync()
    if place:
        bits = src.download(img.dtype, img.shape)
        assert np.array_equal(bits[rows:], img[rows:]) and np.array_equal(bits[:, :8], img[:, :8])
        assert np.array_equal(bits[:, 8 + heads * dh:], img[:, 8 + heads * dh:])
        got = F.from_bf16(bits)[:rows, 8:8 + heads * dh]
    else:
        got, left = read()
        assert left[rows:].all() and left[:, heads * dh:].all()
        got = got[:rows, :heads * dh]
    val = val[:rows, 8:].astype(np.float64).reshape(rows, -1, dh)
    W.check_heads(got.reshape(rows, heads, dh), val[:, :heads], heads, 0, dh, rot, layout, {}, pos[:rows],
                  w if normed else None, q_bf)
    k, off = val[:, heads:heads + kv], np.zeros((rows, kv, dh))
    if normed:
        k, off = R.head_norm(k, w[1], 1e-3)
    k, off = R.turn(k, off, pos[:rows], *R.frequencies(rot), layout == 0)
    check_appended(dev, c, k, off, val[:, heads + kv:], cu, slots)


def check_appended(dev, c, k, off, v, cu, slots):
    """The device's cache is c with K (each within `off`) and V appended: V's bytes, scales of K that its
    largest value can have, codes of K that its values can have, kept codes and zeros exactly."""
    before = [a.copy() for a in (c.k, c.k_exp)]
    c.append(k, v, cu, slots)
    assert np.array_equal(dev.v.download(np.uint8, c.v.shape) & 127 != 0, c.v & 127 != 0)
    assert np.array_equal(O.CODES[dev.v.download(np.uint8, c.v.shape)], O.CODES[c.v])
    assert np.array_equal(dev.v_exp.download(np.uint8, c.v_exp.shape), c.v_exp)
    codes = dev.k.download(np.uint8, c.k.shape)[..., O.places(O.k_at, c.dh)]
    exps = dev.k_exp.download(np.uint8, c.k_exp.shape).astype(np.int64)
    old, old_exps = before[0][..., O.places(O.k_at, c.dh)], before[1].astype(np.int64)
    touched = np.zeros(c.pages, bool)
    differ = total = other = 0
    for b in range(len(cu) - 1):
        r = cu[b]
        while r < cu[b + 1]:
            page, at_ = divmod(int(slots[r]), 64)
            n = min(64 - at_, cu[b + 1] - r)
            touched[page] = True
            x, o = k[r:r + n].transpose(1, 0, 2), off[r:r + n].transpose(1, 0, 2)
            lo, hi = (np.abs(x) - o).clip(0).max((1, 2)), (np.abs(x) + o).max((1, 2))
            e = exps[page]
            floor = old_exps[page] if at_ else 0
            assert (np.maximum(O.exponent(lo), floor) <= e).all() and (e <= np.maximum(O.exponent(hi), floor)).all()
            other += (e != np.maximum(O.exponent(np.abs(x).max((1, 2))), floor)).sum()
            s = O.two(e)[:, None, None]
            got = O.CODES[codes[page][:, at_:at_ + n]]
            value = lambda y: O.CODES[O.encode(np.clip(y / s, -448, 448))]
            assert (value(x - o) <= got).all() and (got <= value(x + o)).all()
            differ += (got != value(x)).sum()
            total += got.size
            kept = np.zeros((c.heads, 64, c.dh))
            if at_:
                kept = O.CODES[O.encode(O.CODES[old[page]] * O.two(127 + floor - e)[:, None, None])]
            rest = np.r_[0:at_, at_ + n:64]
            assert np.array_equal(O.CODES[codes[page][:, rest]], kept[:, rest])
            r += n
    assert np.array_equal(codes[~touched], old[~touched]) and np.array_equal(exps[~touched], old_exps[~touched])
    # values of up to 30 u beside a border, of which there is one in 2^-4 of a value: 2 * 30 u / 2^-4 = 6e-5
    assert differ <= 6e-5 * total + 3 and other <= 1


@pytest.mark.gpu
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("i", range(len(APPENDS)), ids=lambda i: "%dx%d+%d-%dx%d-%d-%d-%d-%s" % APPENDS[i][:9])
def test_rope_append_of_many(gpu_ctx, i, normed):
    append_case(gpu_ctx, i, normed)


# ---- GPU: row offsets that are none ----------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_cache_read_of_row_offsets_that_are_none(gpu_ctx, out):
    """Requests whose offsets fall, begin before the rows or end behind them write nothing; the
    others write exactly their rows."""
    from rembed_amd import tensor as T
    rng = np.random.default_rng(6)
    rows, guard, dh = 40, 30, 64
    c, dev = W.filled(rng, gpu_ctx, 4, 1, dh)
    c.k, c.v = c.k & 0x77, c.v & 0x77                # no NaN
    dev = F.device_cache(gpu_ctx, c)
    table = gpu_ctx.upload(np.array([[0], [1], [2], [3]], I32))
    for cu, done in (([0, 0, 0, 0, rows + 1], []), ([9, 4, 4, 4, 4], []), ([0, -5, 10, 10, 10], []),
                     ([-3, 5, 9, 9, 9], [(1, 5, 9)]), ([2, 7, 7, rows, rows + 20], [(0, 2, 7), (2, 7, rows)]),
                     ([3, 8, rows + 1, rows + 1, rows + 5], [(0, 3, 8)]), ([0, 5, 5, 5, 5], [(0, 0, 5)])):
        buf, read = W.marked(gpu_ctx, rows + guard, 2 * dh, out == "bf16")
        T.CacheRead(gpu_ctx, dev, table, 1, gpu_ctx.upload(np.array(cu, I32)), None, 4, rows, buf, out == "bf16",
                    2 * dh, 0, dh)
        got, left = read()
        written = np.zeros(rows + guard, bool)
        for b, lo, hi in done:
            written[lo:hi] = True
            for x, col in zip(c.rows([b], hi - lo), (0, dh)):
                want = x[:, 0] if out == "f32" else F.bf16(x[:, 0])[0]
                assert np.array_equal(got[lo:hi, col:col + dh], want.astype(np.float32)), cu
        assert left[~written].all(), cu
