"""Edges of the e4m3 operators: memory that was never written, weights far below a row's
largest, tables with pages that are none. Against numpy in 64 bits (fp8_oracle).
"""
import numpy as np
import pytest

import fp8_oracle as O
import test_fp8_operators as F

I32 = np.int32


# ---- GPU: memory that was never written --------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dh,batch,kv,nq,n,gone", [
    # two tiles a workgroup, two halves of the pages: odd numbers of pages, and one alone
    (64, 1, 1, 40, 700, False), (128, 1, 1, 40, 700, False), (256, 1, 1, 40, 700, False),
    (64, 3, 2, 33, 60, False), (128, 3, 2, 33, 60, False), (256, 3, 2, 33, 60, False),
    # four tiles a workgroup, and a page of the table that is none
    (64, 97, 8, 17, 150, True), (128, 97, 8, 17, 150, True), (256, 17, 8, 32, 150, True),
    # few columns
    (128, 3, 2, 1, 700, True), (256, 2, 1, 3, 200, True)])
def test_attention_beside_bytes_never_written(gpu_ctx, dh, batch, kv, nq, n, gone):
    """Page 0 belongs to nobody, and every byte that was never written is 0xFF: NaN as a code and
    as a scale. A page that is none, in the table or behind a range's last, takes no scale
    from there."""
    rng = np.random.default_rng(dh + n)
    blocks = -(-n // 64)
    table = (1 + rng.permutation(batch * blocks).reshape(batch, blocks)).astype(I32)
    c = O.Cache(1 + batch * blocks, kv, dh, fill=0xFF)
    c.k_exp[:], c.v_exp[:] = 255, 255
    cu = np.arange(batch + 1, dtype=I32) * n
    at = np.concatenate([table[b, np.arange(n) // 64].astype(np.int64) * 64 + np.arange(n) % 64
                         for b in range(batch)])
    k, v = rng.standard_normal((2, batch * n, kv, dh))
    c.append(k, v, cu, at)
    assert (c.v_exp[0] == 255).all() and (c.v_exp[1:] != 255).all()
    qcu, lens = np.arange(batch + 1, dtype=I32) * nq, np.full(batch, n, I32)
    q = rng.standard_normal((batch * nq, 2 * kv, dh))
    scale = dh ** -0.5
    want, val = F.attend(gpu_ctx, c, q, "bf16", table, qcu, lens, scale, False, 0, False)
    F.check_attention(c, want, val, table, qcu, lens, scale, False, 0, "bf16", False)
    if gone:  # the first block of the last request: its other keys alone
        bad = table.copy()
        bad[-1, 0] = -1
        got, _ = F.attend(gpu_ctx, c, q, "bf16", bad, qcu, lens, scale, False, 0, False)
        assert np.array_equal(got[:-nq], want[:-nq])
        F.check_attention(c, got[-nq:], val[-nq:], table[-1:, 1:], np.array([0, nq], I32),
                          lens[-1:] - 64, scale, False, 0, "bf16", False)


# ---- GPU: weights far below a row's largest -----------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dh,nq", [(64, 1), (128, 1), (256, 1), (64, 17), (128, 17), (256, 17),
                                   (128, 200)])
@pytest.mark.parametrize("below", [7.0, 10.0, 12.0, 14.0])
@pytest.mark.parametrize("sinks,low,split", [([0], False, False), ([0, 2000], False, True),
                                             ([4095], False, False), ([100], True, False),
                                             ([100], True, True)])
def test_attention_of_weights_that_are_small(gpu_ctx, dh, nq, below, sinks, low, split):
    """A few keys hold nearly all of the weight and no value; thousands lie `below` nats under
    them, with values of one sign, and are all of the result. low: 64 keys before them 96 nats
    further down, so that the reference moves by more than 2^64.

    Every score is a sum of two products that the matrix cores add exactly. A weight p is off by
    half a step of its two codes: 2^-9 of itself, or 2^-21 of the largest weight that its column
    has in its page. A page's products lose STEP of the largest (both codes of P: 1 + 2^-4). The
    fp32 exponents, sums and rescales stay under 2^-15.
    """
    rng = np.random.default_rng(int(below) + nq + dh)
    n = 4133 if split else 4096
    heads = 2
    pages, table, cu, blk, lens, slots = F.batch_of(rng, [n - nq], [nq])
    c = O.Cache(pages, 1, dh)
    k = np.zeros((n, 1, dh))
    k[:, 0, dh - 3] = rng.integers(0, 5, n) / 4
    v = rng.uniform(0.5, 1.5, (n, 1, dh))
    if low:
        k[:64, 0, 1] = -96.0
    for s in sinks:
        k[s, 0, 1], k[s, 0, dh - 3], v[s] = below, 0.0, 0.0
    at = table[0, np.arange(n) // 64].astype(np.int64) * 64 + np.arange(n) % 64
    c.append(k, v, np.array([0, n], I32), at)
    kk, vv = c.rows(table[0], n)
    assert (kk[:, 0, 1] == k[:, 0, 1]).all() and (kk[:, 0, dh - 3] == k[:, 0, dh - 3]).all()
    q = np.zeros((nq, heads, dh))
    q[:, :, 1] = q[:, :, dh - 3] = 1.0
    got, _ = F.attend(gpu_ctx, c, q, "bf16", table, cu, lens, 1.0, False, 0, False,
                      max_len=n if split else 64)
    s = kk[:, 0, 1] + kk[:, 0, dh - 3]
    p = np.exp(s - s.max())
    p /= p.sum()
    top = np.repeat(np.maximum.reduceat(p, np.arange(0, n, 64)), 64)[:n]
    want = p @ vv[:, 0]
    off = np.maximum(2.0 ** -9 * p, 2.0 ** -21 * top) @ np.abs(vv[:, 0])
    drop = np.maximum.reduceat(p[:, None] * np.abs(vv[:, 0]), np.arange(0, n, 64), 0).sum(0)
    tol = off + F.STEP * (1 + 2.0 ** -4) * drop + 2.0 ** -15 * want
    assert (tol <= 2.0 ** -5 * want).all()  # it says something about the small weights
    assert (np.abs(got - want) <= tol).all(), np.abs(got / want - 1).max()


@pytest.mark.gpu
@pytest.mark.parametrize("dh,nq", [(64, 1), (128, 20), (256, 200)])
@pytest.mark.parametrize("size", [20, 23, 24, 25, 26, 27, 28, 29, 60, 100])
def test_attention_of_scores_of_any_size(gpu_ctx, dh, nq, size):
    """Scores of 2^size and half of it, up and down from page to page: the keys of the larger
    ones share the weight, each p the same number within 2^-9 of 1 / their count."""
    rng = np.random.default_rng(size)
    n = 64 * 9 + 11
    pages, table, cu, blk, lens, slots = F.batch_of(rng, [max(0, n - nq)], [nq])
    c = O.Cache(pages, 1, dh)
    k = np.zeros((n, 1, dh))
    one = rng.integers(0, 3, n) == 0
    one[:64] = False  # the first page is far below the others
    k[:, 0, 1] = np.where(one, 2.0, 1.0) * 2.0 ** (size // 2 - 1)
    v = rng.standard_normal((n, 1, dh))
    at = table[0, np.arange(n) // 64].astype(np.int64) * 64 + np.arange(n) % 64
    c.append(k, v, np.array([0, n], I32), at)
    kk, vv = c.rows(table[0], n)
    assert (kk == k).all()
    q = np.zeros((nq, 2, dh))
    q[:, :, 1] = 2.0 ** (size - size // 2)
    got, _ = F.attend(gpu_ctx, c, q, "bf16", table, cu, lens, 1.0, False, 0, False)
    want, mag = vv[one, 0].mean(0), np.abs(vv[one, 0]).mean(0)
    tol = (2.0 ** -9 + F.STEP * (1 + 2.0 ** -4)) * mag + 2.0 ** -20
    assert (np.abs(got - want) <= tol).all()


# ---- GPU: rows without a page ---------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dh", [64, 256])
@pytest.mark.parametrize("none", [-1, 1 << 20])
def test_append_behind_a_page_that_is_none(gpu_ctx, dh, none):
    """A block whose page is negative or behind the cache's last is skipped; the request's
    other blocks are written, from its first row of theirs on."""
    past, fresh = [10, 70, 63, 5, 0, 127], [54 + 64 + 9, 3, 1, 60, 130, 66]
    rng = np.random.default_rng(dh)
    heads, pages = 2, 16
    table = np.full((6, 4), none, I32)
    table[1, :2] = [0, 1]
    free = rng.permutation(np.arange(2, pages)).astype(I32)
    n = sum(fresh)
    cu, blk, lens, slots, _, status = O.plan(past, fresh, free, table, n)
    assert status[0] == 0
    table[4, 1] = none  # a middle block of request 4 as well
    first = int(cu[4])
    slots[first + 64:first + 128] = -1 if none < 0 else none * 64 + np.arange(64)
    c = O.Cache(pages, heads, dh)
    dev = F.device_cache(gpu_ctx, c)
    k, v = rng.standard_normal((2, n, heads, dh))
    k, v = F.append(gpu_ctx, dev, k, v, "bf16", cu, blk, slots)
    c.append(k, v, cu, slots)
    assert (c.k_exp[table[0, 1]] != 200).all()  # the second block of request 0 was written
    F.same_cache(dev, c)


# ---- GPU: more rows than a call was told of -------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dh,heads,max_q,past", [
    (64, 2, 2, 4000), (128, 4, 1, 4000), (256, 2, 3, 2000),  # few columns, key ranges split
    (64, 2, 7, 200), (128, 2, 40, 4000), (256, 2, 70, 300)])
def test_attention_of_more_rows_than_max_q(gpu_ctx, dh, heads, max_q, past):
    """A request's first max_q rows are what they are in a call of that many rows' room; the
    others, and the bytes behind the scratch, are left as they were."""
    from rembed_amd import tensor as T
    rng = np.random.default_rng(dh + max_q)
    fresh = [max_q + 9, max_q, max_q + 90, 1]
    pages, table, cu, blk, lens, slots = F.batch_of(rng, [past] * 4, fresh)
    c = O.Cache(pages, 1, dh)
    acu = np.concatenate([[0], np.cumsum(lens)]).astype(I32)
    at = np.concatenate([table[b, np.arange(n) // 64].astype(np.int64) * 64 + np.arange(n) % 64
                         for b, n in enumerate(lens)])
    k, v = rng.standard_normal((2, len(at), 1, dh))
    c.append(k, v, acu, at)
    dev, scale = F.device_cache(gpu_ctx, c), dh ** -0.5
    img, val = F.typed(rng.standard_normal((int(cu[-1]), heads * dh)), "bf16")
    q = val.astype(np.float64).reshape(-1, heads, dh)
    need = T.cache_attention_scratch(4, max_q, int(max(lens)), heads, 1, dh)
    assert (need > 0) == (past > 1000)
    scratch = gpu_ctx.upload(np.full(need + (1 << 20), 0x5A, np.uint8))
    out = gpu_ctx.upload(np.full((int(cu[-1]), heads * dh), 55, np.float32))
    T.CacheAttention(gpu_ctx, out, False, heads * dh, gpu_ctx.upload(img), True, heads * dh, 0, dev,
                     gpu_ctx.upload(table), table.shape[1], gpu_ctx.upload(cu),
                     gpu_ctx.upload(lens), 4, max_q, int(max(lens)), heads, scale, True, 0,
                     scratch, need)
    gpu_ctx.sync()
    assert (scratch.download(np.uint8, (need + (1 << 20),))[need:] == 0x5A).all()
    got = out.download(np.float32, (int(cu[-1]), heads * dh))
    for b, n in enumerate(fresh):
        first = slice(cu[b], cu[b] + min(n, max_q))
        assert (got[first.stop:cu[b + 1]] == 55).all()
        kk, vv = c.rows(table[b], int(lens[b]))
        want, mag, top = O.attention(q[cu[b]:cu[b + 1]], kk, vv, scale, True, 0)
        rows = first.stop - first.start
        ds = scale * top * (dh / 64 * F.STEP * (1 + 2.0 ** -4))
        tol = (F.BF16 + F.STEP * (1 + 2.0 ** -4) + 2 * ds) * mag[:rows] + 1e-6
        assert (np.abs(got[first].reshape(rows, heads, dh) - want[:rows]) <= tol).all()


# ---- linears whose output lies on their rows ----------------------------------------------

def test_rows_that_share_bytes():
    import ctypes

    from rembed_amd import _lib
    f = ctypes.CDLL(_lib.LIB_PATH)._ZN2rh12rows_overlapEPKvmmS1_mmi
    P, S = ctypes.c_void_p, ctypes.c_size_t
    f.argtypes, f.restype = [P, S, S, P, S, S, ctypes.c_int], ctypes.c_bool

    def brute(a, wa, sa, b, wb, sb, m):
        rows = lambda x, w, s: {x + r * s + i for r in range(m) for i in range(w)}
        return bool(rows(a, wa, sa) & rows(b, wb, sb))

    rng = np.random.default_rng(0)
    for _ in range(3000):
        m, wa, wb = rng.integers(1, 5), rng.integers(1, 9), rng.integers(1, 9)
        sa = sb = max(wa, wb) + int(rng.integers(0, 9))
        a, b = (4096 + int(x) for x in rng.integers(0, 60, 2))
        if rng.random() < 0.5:
            sa, sb = wa + int(rng.integers(0, 9)), wb + int(rng.integers(0, 9))
        want, got = brute(a, wa, sa, b, wb, sb, m), f(a, wa, sa, b, wb, sb, int(m))
        # rows side by side exactly, others never too few
        assert got == want if sa == sb and abs(b - a) < sa else got >= want
    assert not f(4096, 8, 24, 4096 + 8, 16, 24, 9) and f(4096, 8, 24, 4096 + 7, 16, 24, 9)
    assert not f(4096 + 16, 8, 24, 4096, 16, 24, 9) and f(4096, 8, 8, 4096, 8, 8, 9)
    assert not f(4096, 8, 8, 4096, 8, 8, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(1, 4096, 4096), (16, 1024, 1024), (5, 3584, 3584), (40, 640, 640),
                                   (64, 512, 512), (300, 768, 768)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_linear_over_its_own_rows(gpu_ctx, m, k, n, dtype):
    """dst is a: the same bits as into a buffer of its own."""
    from rembed_amd import tensor as T
    rng = np.random.default_rng(m + k)
    img, _ = F.typed(rng.standard_normal((m, k)), dtype)
    pb = T.PackFP8(gpu_ctx, rng.standard_normal((n, k)).astype(np.float32), k, n)
    bf, ldq = dtype == "bf16", T.ldq_fp8(k)
    qa, sa = gpu_ctx.alloc(m * ldq), gpu_ctx.alloc(T.fp8_scale_bytes(m, k))
    a, out = gpu_ctx.upload(img), gpu_ctx.alloc(img.nbytes)
    T.LinearFP8(gpu_ctx, out, bf, n, a, bf, k, pb, m, 0, qa, ldq, sa)
    want = out.download(img.dtype, (m, n))
    T.LinearFP8(gpu_ctx, a, bf, n, a, bf, k, pb, m, 0, qa, ldq, sa)
    assert np.array_equal(a.download(img.dtype, (m, n)), want)
    if dtype == "f32":
        a = gpu_ctx.upload(img)
        T.Linear(gpu_ctx, a, a, pb, m)
        assert np.array_equal(a.download(img.dtype, (m, n)), want)


# ---- GPU: rows of nearly 2^31 values ---------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("k", [0x7FFFFF00, 0x7FFFFF00 - 3, 0x7FFFFE00])
def test_quantize_the_longest_rows(gpu_ctx, k):
    """One bf16 row of up to the most values that a call takes: its last blocks."""
    from rembed_amd import _lib
    from rembed_amd import tensor as T
    ldq, tail = T.ldq_fp8(k), 1000
    rng = np.random.default_rng(1)
    val, bits = F.bf16(rng.standard_normal(tail) * np.exp(rng.uniform(-4, 4, tail)))
    a, qa = gpu_ctx.alloc(k * 2), gpu_ctx.alloc(ldq)
    sa = gpu_ctx.alloc(T.fp8_scale_bytes(1, k))
    _lib.check(_lib.lib.rh_memcpy_h2d(gpu_ctx.h, a.ptr + (k - tail) * 2, bits.ctypes.data, tail * 2))
    T.QuantizeRowsFP8(gpu_ctx, a, True, k, 1, k, qa, ldq, sa)
    codes, exps = np.empty(512, np.uint8), np.empty(4 * 128, np.uint8)
    _lib.check(_lib.lib.rh_memcpy_d2h(gpu_ctx.h, codes.ctypes.data, qa.ptr + ldq - 512, 512))
    _lib.check(_lib.lib.rh_memcpy_d2h(gpu_ctx.h, exps.ctypes.data, sa.ptr + ldq - 512, 512))
    last = np.zeros(512)
    last[:512 - (ldq - k)] = val[tail - (512 - (ldq - k)):]
    want, e, _ = O.quantize_rows(last[None])
    assert np.array_equal(exps.reshape(4, 128)[:, 0], e[0])
    assert np.array_equal(O.CODES[codes], O.CODES[want[0]])


# ---- the rule that reads pages past the L2 --------------------------------------------------

def test_pages_read_past_the_l2():
    """Only where pages that exist, of at most all requests, exceed 256 MiB: texts behind a
    shared beginning do not make them more than the cache holds."""
    import ctypes

    from rembed_amd import _lib
    f = ctypes.CDLL(_lib.LIB_PATH)._ZN2rh13cache_streamsExiiii
    f.argtypes, f.restype = [ctypes.c_longlong] + [ctypes.c_int] * 4, ctypes.c_bool
    assert f(128, 48, 4000, 8, 128)            # 48 texts of up to 8192: 524 MB of pages
    assert not f(11, 256, 266, 8, 128)         # 256 queries behind one prefix of ten pages
    assert f(11, 256, 2816, 8, 128)            # each with ten of its own
    page = 64 * 8 * 128 * 2
    assert not f(1, 2 ** 28 // page, 1 << 20, 8, 128) and f(1, 2 ** 28 // page + 1, 1 << 20, 8, 128)
    assert not f(2 ** 25, 2 ** 20, 0, 8, 128) and f(2 ** 25, 2 ** 20, 2 ** 31 - 1, 64, 256)


@pytest.mark.gpu
@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("nq", [1, 5])
def test_attention_over_a_cache_that_is_large(gpu_ctx, dh, nq):
    """Few columns over a cache of more than 256 MiB, pages read past the L2, some of them shared,
    from all over it; bytes that were never written lie between."""
    from rembed_amd import tensor as T
    rng = np.random.default_rng(dh + nq)
    past, fresh, heads = [700, 64, 0, 1300], [nq, 1, nq, nq], 2
    pages, table, cu, blk, lens, slots = F.batch_of(rng, past, fresh)
    many = 2 ** 28 // (heads * 64 * dh * 2) + 100
    where = rng.choice(many, pages, replace=False).astype(I32)
    c, dev = O.Cache(pages, heads, dh), T.KVCache(gpu_ctx, many, heads, dh)
    acu = np.concatenate([[0], np.cumsum(lens)]).astype(I32)
    ablk = np.concatenate([[0], np.cumsum(-(-np.asarray(lens) // 64))]).astype(I32)
    at = np.concatenate([table[b, np.arange(n) // 64].astype(np.int64) * 64 + np.arange(n) % 64
                         for b, n in enumerate(lens)])
    k, v = rng.standard_normal((2, len(at), heads, dh))
    k, v = F.append(gpu_ctx, dev, k, v, "bf16", acu, ablk,
                    where[at // 64].astype(np.int64) * 64 + at % 64)
    c.append(k, v, acu, at)
    table[1, 0] = table[0, 0]  # a shared page
    dev.heads = heads
    q = rng.standard_normal((int(cu[-1]), 4, dh))
    for max_len in (int(max(lens)), 3_000_000):
        for dtype, out_bf16 in (("bf16", True), ("f32", False)):
            got, val = F.attend(gpu_ctx, dev, q, dtype, where[table], cu, lens, dh ** -0.5, True, 0,
                                out_bf16, max_len=max_len)
            F.check_attention(c, got, val, table, cu, lens, dh ** -0.5, True, 0, dtype, out_bf16)
