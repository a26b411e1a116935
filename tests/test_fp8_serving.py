"""The e4m3 serving path as a decoder layer runs it: linears, block tables, the cache and its
attention behind each other, step after step, recorded as HIP graphs, on two contexts at once,
and at sizes where other tiles and offsets past 32 bits are used. Against numpy in 64 bits
(fp8_oracle); tolerances as in test_fp8_operators.
"""
import ctypes
import threading

import numpy as np
import pytest

import fp8_oracle as O
import test_fp8_operators as F

pytestmark = pytest.mark.gpu
I32 = np.int32


def close_linear(got, x, wv, bias, act, out_bf16):
    """got against act(e4m3(x) . wv + bias): the norm's bound (NORM, the result's rounding),
    and a step's largest product by elements."""
    _, _, xv = O.quantize_rows(x.astype(np.float64))
    y = xv @ wv.T
    z = y if bias is None else y + bias
    want = F.act_of(z, act)
    drop = np.zeros(y.shape)
    for s in range(0, x.shape[1], 64):
        drop += F.STEP * np.outer(np.abs(xv[:, s:s + 64]).max(1), np.abs(wv[:, s:s + 64]).max(1))
    tol = 1.13 * drop + 2.0 ** -18 * (np.abs(want) + np.abs(xv) @ np.abs(wv).T) + 1e-30
    tol += (F.BF16 if out_bf16 else 0) * (np.abs(want) + 1.13 * drop)
    assert (np.abs(got - want) <= tol).all()
    if np.linalg.norm(want):
        norm = np.linalg.norm(got - want) / np.linalg.norm(want)
        assert norm <= (F.BF16 if out_bf16 else 0) + 1.13 * F.NORM * max(
            1.0, np.linalg.norm(y) / np.linalg.norm(want)), norm


class Layer:
    """q|k|v, attention's output and a gated MLP of one decoder layer, with its cache."""

    def __init__(self, ctx, hidden, heads, kv, dh, inter, batch, pages, ldt, rows, max_len, seed=0):
        from rembed_amd import tensor as T
        rng = np.random.default_rng(seed)
        self.ctx, self.hidden, self.heads, self.kv = ctx, hidden, heads, kv
        self.dh, self.inter = dh, inter
        self.batch, self.rows, self.max_len = batch, rows, max_len
        self.width = (heads + 2 * kv) * dh

        def weight(n, k):
            return (rng.standard_normal((n, k)) * (1.5 / k ** 0.5)).astype(np.float32)

        self.w = {"qkv": weight(self.width, hidden), "o": weight(hidden, heads * dh),
                  "gate": weight(inter, hidden), "up": weight(inter, hidden),
                  "down": weight(hidden, inter)}
        self.b = rng.standard_normal(self.width).astype(np.float32)
        self.pw = {"qkv": T.PackFP8(ctx, self.w["qkv"], hidden, self.width, self.b),
                   "o": T.PackFP8(ctx, self.w["o"], heads * dh, hidden),
                   "mlp": T.PackedGated(ctx, 3, self.w["gate"], self.w["up"], hidden, inter),
                   "down": T.PackFP8(ctx, self.w["down"], inter, hidden)}
        self.val = {n: O.quantize_weight(x.astype(np.float64))[2] for n, x in self.w.items()}
        # the device's buffers of a step
        self.past, self.fresh = ctx.alloc(batch * 4), ctx.alloc(batch * 4)
        self.free, self.n_free = ctx.alloc(pages * 4), pages
        self.ldt = ldt
        self.table = ctx.upload(np.full((batch, ldt), -1, I32))
        self.cu, self.blocks = ctx.alloc(batch * 4 + 4), ctx.alloc(batch * 4 + 4)
        self.lens, self.status = ctx.alloc(batch * 4), ctx.alloc(16)
        self.slots, self.pos = ctx.alloc(rows * 8), ctx.alloc(rows * 4)
        k = max(hidden, heads * dh, inter)
        self.qa, self.sa = ctx.alloc(rows * T.ldq_fp8(k)), ctx.alloc(T.fp8_scale_bytes(rows, k))
        self.x, self.qkv = ctx.alloc(rows * hidden * 2), ctx.alloc(rows * self.width * 2)
        self.att, self.o = ctx.alloc(rows * heads * dh * 2), ctx.alloc(rows * hidden * 2)
        self.mid, self.y = ctx.alloc(rows * inter * 2), ctx.alloc(rows * hidden * 4)
        self.oracle = O.Cache(pages, kv, dh, fill=0x55)
        self.cache = F.device_cache(ctx, self.oracle)
        self.need = max(T.cache_attention_scratch(batch, n, max_len, heads, kv, dh)
                        for n in range(1, rows + 1))
        self.scratch = ctx.alloc(self.need)

    def give(self, past, fresh, free, x):
        """The step's inputs to the device."""
        from rembed_amd import _lib
        for buf, a in ((self.past, np.array(past, I32)), (self.fresh, np.array(fresh, I32)),
                       (self.free, np.array(free, I32)), (self.x, np.ascontiguousarray(x))):
            _lib.check(_lib.lib.rh_memcpy_h2d(self.ctx.h, buf.ptr, a.ctypes.data, a.nbytes))

    def step(self, m, n_free, max_q, scratch=None):
        """Enqueues a step of m rows."""
        from rembed_amd import tensor as T
        c, h = self.ctx, self.hidden
        T.CachePlan(c, self.past, self.fresh, self.batch, self.free, n_free, self.table, self.ldt,
                    self.cu, self.blocks, self.lens, self.slots, self.pos, m, self.status)

        def linear(dst, bf, ldd, src, k, w, act):
            T.LinearFP8(c, dst, bf, ldd, src, True, k, w, m, act, self.qa, T.ldq_fp8(k), self.sa)

        linear(self.qkv, True, self.width, self.x, h, self.pw["qkv"], 0)
        hd = self.heads * self.dh
        T.CacheAppend(c, self.cache, self.qkv, True, self.width, hd, hd + self.kv * self.dh, self.cu,
                      self.blocks, self.slots, self.batch, m)
        T.CacheAttention(c, self.att, True, hd, self.qkv, True, self.width, 0, self.cache, self.table,
                         self.ldt, self.cu, self.lens, self.batch, max_q, self.max_len, self.heads,
                         self.dh ** -0.5, True, 0, scratch or self.scratch, self.need)
        linear(self.o, True, h, self.att, hd, self.pw["o"], 0)
        linear(self.mid, True, self.inter, self.o, h, self.pw["mlp"], 2)
        linear(self.y, False, h, self.mid, self.inter, self.pw["down"], 0)

    def got(self, m):
        self.ctx.sync()
        bf = lambda b, n: F.from_bf16(b.download(np.uint16, (m, n)))
        return {"qkv": bf(self.qkv, self.width), "att": bf(self.att, self.heads * self.dh),
                "o": bf(self.o, self.hidden), "mid": bf(self.mid, self.inter),
                "y": self.y.download(np.float32, (m, self.hidden))}


def batch_x(rng, m, hidden):
    v, bits = F.bf16(rng.standard_normal((m, hidden)))
    return v, bits


@pytest.mark.parametrize("heads,kv,dh", [(4, 2, 64), (4, 4, 128), (3, 1, 256)])
def test_decoder_layer_steps(gpu_ctx, heads, kv, dh):
    """Prompts, then tokens, one request joining late and one pausing: every operator's output
    against 64 bits of what it was given, the cache's bytes after every step."""
    L = Layer(gpu_ctx, 192, heads, kv, dh, 272, 4, 40, 9, 400, 600)
    rng = np.random.default_rng(dh)
    order = rng.permutation(40).astype(I32)
    past, taken = np.zeros(4, int), 0
    table = np.full((4, 9), -1, I32)
    for fresh in ([130, 5, 0, 64], [1, 1, 0, 1], [1, 60, 190, 1], [1, 1, 1, 0], [3, 1, 2, 70],
                  [1, 1, 1, 1]):
        m = sum(fresh)
        x, bits = batch_x(rng, m, 192)
        free = order[taken:]
        L.give(past, fresh, free, bits)
        L.step(m, len(free), max(fresh))
        cu, blocks, lens, slots, pos, status = O.plan(past, fresh, free, table, m)
        got = L.got(m)
        assert np.array_equal(L.slots.download(np.int64, (m,)), slots)
        assert L.status.download(I32, (4,)).tolist() == status
        assert np.array_equal(L.table.download(I32, table.shape), table)
        close_linear(got["qkv"], x, L.val["qkv"], L.b, 0, True)
        r = got["qkv"].astype(np.float64)
        q = r[:, :heads * dh].reshape(m, heads, dh)
        k = r[:, heads * dh:(heads + kv) * dh].reshape(m, kv, dh)
        v = r[:, (heads + kv) * dh:].reshape(m, kv, dh)
        L.oracle.append(k, v, cu, slots)
        F.same_cache(L.cache, L.oracle)
        F.check_attention(L.oracle, got["att"].reshape(m, heads, dh).astype(np.float64), q, table,
                          cu, lens, dh ** -0.5, True, 0, "bf16", True)
        close_linear(got["o"], got["att"], L.val["o"], None, 0, True)
        _, _, ov = O.quantize_rows(got["o"].astype(np.float64))
        want = F.gated(ov @ L.val["gate"].T, ov @ L.val["up"].T, 2)
        assert np.linalg.norm(got["mid"] - want) <= (F.BF16 + 3 * F.NORM) * np.linalg.norm(want)
        close_linear(got["y"], got["mid"], L.val["down"], None, 0, False)
        past = past + fresh
        taken += status[2]


class Recorded:
    """What `enqueue` puts on the context's stream, as a HIP graph."""

    def __init__(self, ctx, enqueue):
        from rembed_amd import _lib
        self.hip, self.stream = _lib.hip_runtime(), ctypes.c_void_p(ctx.stream)
        graph, self.exec = ctypes.c_void_p(), ctypes.c_void_p()
        self.ok(self.hip.hipStreamBeginCapture(self.stream, 1))
        enqueue()
        self.ok(self.hip.hipStreamEndCapture(self.stream, ctypes.byref(graph)))
        self.ok(self.hip.hipGraphInstantiate(ctypes.byref(self.exec), graph, None, None,
                                             ctypes.c_size_t(0)))
        self.ok(self.hip.hipGraphDestroy(graph))

    @staticmethod
    def ok(status):
        assert status == 0, status

    def replay(self):
        self.ok(self.hip.hipGraphLaunch(self.exec, self.stream))

    def close(self):
        self.ok(self.hip.hipGraphExecDestroy(self.exec))


@pytest.mark.parametrize("fresh,dh", [([1, 1, 1], 128), ([40, 33, 50], 64), ([20, 1, 70], 256)])
def test_recorded_steps(gpu_ctx, fresh, dh):
    """Two layers' steps recorded as graphs that share one scratch, replayed in turn, with eager
    steps of other sizes and synchronizations in between: the bits of steps launched one by one."""
    past0 = [700, 130, 64]
    layers = [Layer(gpu_ctx, 128, 4, 2, dh, 144, 3, 60, 20, 240, 1200, seed=s) for s in (1, 2, 1, 2)]
    rec, eager = layers[:2], layers[2:]
    for a in layers[1:]:
        assert a.need == layers[0].need > 0  # ranges are joined
    m = sum(fresh)
    order = np.random.default_rng(5).permutation(60).astype(I32)
    rng = np.random.default_rng(6)
    past = np.zeros(3, int)
    taken = 0
    for first in (past0, fresh):  # the prompts in pieces, eagerly, on all four
        todo = np.array(first)
        while todo.any():
            f = np.minimum(todo, 80)
            _, bits = batch_x(rng, int(f.sum()), 128)
            for a in layers:
                a.give(past, f, order[taken:], bits)
                a.step(int(f.sum()), 60 - taken, 80)
                gpu_ctx.sync()
            taken += int(layers[0].status.download(I32, (4,))[2])
            past, todo = past + f, todo - f
    graphs = [Recorded(gpu_ctx, lambda a=a: a.step(m, 60, max(fresh), layers[0].scratch)) for a in rec]
    for turn in range(5):
        f = np.array(fresh)
        _, bits = batch_x(rng, m, 128)
        free = np.resize(order[taken:], 60)  # what is behind the first ones is not taken
        for a in layers:
            a.give(past, f, free, bits)
        for g in graphs:
            g.replay()
        if turn % 2:
            gpu_ctx.sync()
        for a in eager:
            a.step(m, 60, max(fresh))
        for a, b in zip(rec, eager):
            x, y = a.got(m), b.got(m)
            for name in x:
                assert np.array_equal(x[name].view(np.uint32), y[name].view(np.uint32)), (turn, name)
            for name in ("k", "v", "k_exp", "v_exp"):
                s = (getattr(a.cache, name).nbytes,)
                assert np.array_equal(getattr(a.cache, name).download(np.uint8, s),
                                      getattr(b.cache, name).download(np.uint8, s)), (turn, name)
        assert layers[0].status.download(I32, (4,))[0] == 0
        taken += int(layers[0].status.download(I32, (4,))[2])
        past = past + f
    for g in graphs:
        g.close()


def test_two_contexts_at_once():
    """Steps on two contexts from two threads: what each gives alone."""
    from rembed_amd import tensor as T

    def work(ctx, seed, out):
        L = Layer(ctx, 256, 8, 2, 128, 272, 4, 60, 20, 600, 1300, seed=seed)
        rng = np.random.default_rng(seed)
        past, taken = np.zeros(4, int), 0
        for fresh in ([150, 90, 3, 200], [1, 1, 1, 1], [1, 140, 1, 1], [1, 1, 1, 1], [1, 1, 1, 1]):
            _, bits = batch_x(rng, sum(fresh), 256)
            L.give(past, fresh, np.arange(taken, 60), bits)
            L.step(sum(fresh), 60 - taken, max(fresh))
            out.append(L.got(sum(fresh)))
            taken += int(L.status.download(I32, (4,))[2])
            past = past + fresh

    with T.Context(0) as c1, T.Context(0) as c2:
        alone, both = ([], []), ([], [])
        work(c1, 1, alone[0])
        work(c2, 2, alone[1])
        threads = [threading.Thread(target=work, args=(c, s, o))
                   for c, s, o in ((c1, 1, both[0]), (c2, 2, both[1]))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for a, b in zip(alone, both):
            assert len(a) == len(b) == 5
            for x, y in zip(a, b):
                for name in x:
                    assert np.array_equal(x[name].view(np.uint32), y[name].view(np.uint32)), name


@pytest.mark.parametrize("m,k,n,dtype", [
    (1, 512, 272, "f32"), (16, 1280, 144, "f32"), (17, 640, 272, "bf16"), (40, 2560, 400, "bf16"),
    (130, 1024, 144, "f32"), (250, 250, 256, "bf16"), (64, 301, 144, "f32"), (5, 3584, 144, "f32"),
    (16, 1000, 8192, "bf16")])
def test_linear_of_rows_made_on_the_way(gpu_ctx, m, k, n, dtype):
    """Few rows are made e4m3 inside the product: the bits of quantizing them first, whatever
    the stride and alignment by which they are read."""
    from rembed_amd import tensor as T
    rng = np.random.default_rng(m + k)
    x = rng.standard_normal((m, k)) * np.exp(rng.uniform(-9, 9, (m, 1)))
    x[0, : k // 2] = 0.0
    img, val = F.typed(x, dtype)
    b = rng.standard_normal(n).astype(np.float32)
    w = (rng.standard_normal((n, k)) / k ** 0.5).astype(np.float32)
    pb = T.PackFP8(gpu_ctx, w, k, n, b)
    ldq, bf = T.ldq_fp8(k), dtype == "bf16"
    qa, sa = gpu_ctx.alloc(m * ldq), gpu_ctx.alloc(T.fp8_scale_bytes(m, k))
    dst = gpu_ctx.alloc(m * n * 4)
    T.QuantizeRowsFP8(gpu_ctx, gpu_ctx.upload(img), bf, k, m, k, qa, ldq, sa)
    T.MatMulFP8(gpu_ctx, dst, False, n, qa, ldq, sa, pb, m, 1)
    want = dst.download(np.float32, (m, n))
    close_linear(want, val, O.quantize_weight(w.astype(np.float64))[2], b, 1, False)
    for lda, front in ((k, 0), (k + 3, 0), ((k + 15) // 8 * 8, 0), ((k + 15) // 8 * 8, 1)):
        rows = np.full((m, lda), 0x7FC0 if bf else np.nan, img.dtype)  # NaN beside the rows
        rows[:, :k] = img
        d = gpu_ctx.upload(np.concatenate([np.zeros(front, img.dtype), rows.ravel(),
                                           np.zeros(8, img.dtype)]))
        at = Part(gpu_ctx, d.ptr + front * img.itemsize, 0)
        T.LinearFP8(gpu_ctx, dst, False, n, at, bf, lda, pb, m, 1, qa, ldq, sa)
        assert np.array_equal(dst.download(np.float32, (m, n)).view(np.uint32),
                              want.view(np.uint32)), (lda, front)


# sizes by which tiles of 64 x 64, 128 x 128, 128 x 256 and 256 x 256 are chosen
@pytest.mark.parametrize("m,k,n", [(1100, 200, 1008), (1500, 384, 2000), (2050, 256, 3008),
                                   (4097, 320, 2064), (4000, 136, 4000)])
def test_linears_of_many_rows(gpu_ctx, m, k, n):
    from rembed_amd import tensor as T
    rng = np.random.default_rng(m + n)
    x = rng.standard_normal((m, k)) * np.exp(rng.standard_normal((m, 1)))
    w = (rng.standard_normal((n, k)) / k ** 0.5).astype(np.float32)
    b = rng.standard_normal(n).astype(np.float32)
    _, _, wv = O.quantize_weight(w.astype(np.float64))
    for dtype, bias, act, out_bf16 in (("bf16", None, 0, True), ("f32", b, 0, False)):
        img, val = F.typed(x, dtype)
        pb = T.PackFP8(gpu_ctx, w, k, n, bias)
        got = F.run_linear(gpu_ctx, pb, img, dtype == "bf16", m, k, n, act, out_bf16, n + 4)
        close_linear(got, val, wv, bias, act, out_bf16)


@pytest.mark.parametrize("m,k,i", [(1300, 256, 640), (2050, 200, 1504), (4100, 128, 1040)])
def test_gated_linears_of_many_rows(gpu_ctx, m, k, i):
    from rembed_amd import tensor as T
    rng = np.random.default_rng(m + i)
    x = rng.standard_normal((m, k))
    g, u = (rng.standard_normal((2, i, k)) / k ** 0.5).astype(np.float32)
    pb = T.PackedGated(gpu_ctx, 3, g, u, k, i)
    gv, uv = (O.quantize_weight(w.astype(np.float64))[2] for w in (g, u))
    for dtype, out_bf16 in (("f32", False), ("bf16", True)):
        img, val = F.typed(x, dtype)
        _, _, xv = O.quantize_rows(val.astype(np.float64))
        want = F.gated(xv @ gv.T, xv @ uv.T, 2)
        got = F.run_linear(gpu_ctx, pb, img, dtype == "bf16", m, k, i, 2, out_bf16, i)
        assert np.linalg.norm(got - want) <= ((F.BF16 if out_bf16 else 0) + 3 * F.NORM) * \
            np.linalg.norm(want)


def test_linear_of_rows_past_32_bits(gpu_ctx):
    """2^25 + 300 rows of one value: codes of more than 2^32 bytes, more rows than a launch
    of the quantizer takes."""
    from rembed_amd import tensor as T
    m, n = (1 << 25) + 300, 16
    x = np.random.default_rng(1).standard_normal((m, 1)).astype(np.float32)
    w = np.arange(1, 17, dtype=np.float32)[:, None]
    _, _, wv = O.quantize_weight(w.astype(np.float64))
    pb = T.PackFP8(gpu_ctx, w, 1, n)
    d, dst = gpu_ctx.upload(x), gpu_ctx.alloc(m * n * 2)
    qa, sa = gpu_ctx.alloc(m * 128), gpu_ctx.alloc(T.fp8_scale_bytes(m, 1))
    T.LinearFP8(gpu_ctx, dst, True, n, d, False, 1, pb, m, 0, qa, 128, sa)
    bits = dst.download(np.uint16, (m, n))
    at = np.concatenate([np.arange(0, m, 997), np.arange(1 << 24, (1 << 24) + 500),
                         np.arange((1 << 25) - 500, m)])
    _, _, xv = O.quantize_rows(x[at].astype(np.float64))
    want = xv @ wv.T
    assert (np.abs(F.from_bf16(bits[at]) - want) <= F.BF16 * 1.01 * np.abs(want) + 1e-30).all()


# heads, kv heads, dh, past, fresh, causal, window: four tiles per workgroup
WIDE = [
    (32, 16, 64, [100], [1600], True, 0), (32, 16, 64, [100] * 5, [300, 7, 290, 0, 299], True, 200),
    (16, 8, 128, [0, 65, 300], [1050, 1060, 1], True, 0), (8, 4, 128, [500], [6300], True, 300),
    (8, 2, 256, [1800, 3], [300, 299], True, 0), (8, 2, 256, [1000] * 4, [600, 1, 65, 610], False, 100),
]


@pytest.mark.parametrize("case", WIDE, ids=lambda c: "%dx%dx%d-%d" % (c[0], c[1], c[2], len(c[3])))
def test_attention_of_many_columns(gpu_ctx, case):
    heads, kv, dh, past, fresh, causal, window = case
    rng = np.random.default_rng(dh + len(past))
    pages, table, cu, blk, lens, slots = F.batch_of(rng, past, fresh)
    c = O.Cache(pages, kv, dh)
    acu = np.concatenate([[0], np.cumsum(lens)]).astype(I32)
    asl = np.concatenate([table[b, np.arange(n) // 64].astype(np.int64) * 64 + np.arange(n) % 64
                          for b, n in enumerate(lens)])
    k, v = rng.standard_normal((2, len(asl), kv, dh))
    c.append(k, v, acu, asl)
    q = rng.standard_normal((int(cu[-1]), heads, dh))
    got, val = F.attend(gpu_ctx, c, q, "bf16", table, cu, lens, dh ** -0.5, causal, window, True, pad=8)
    # rows here and there: the last of a tile, the first, the last
    for b, n in enumerate(lens):
        nq = cu[b + 1] - cu[b]
        kk, vv = c.rows(table[b], int(n))
        for r in sorted({0, 1, 15, 16, 31, 32, 63, 64, 127, 128, 255, nq // 2, nq - 2, nq - 1}):
            if not 0 <= r < nq:
                continue
            i = n - nq + r
            lo, hi = 0, n
            if causal:
                hi = i + 1
            if window:
                lo, hi = max(lo, i - window + 1), min(hi, i + window)
            want, mag, top = O.attention(val[cu[b] + r:cu[b] + r + 1], kk[lo:hi], vv[lo:hi],
                                         dh ** -0.5, False, 0)
            ds = dh ** -0.5 * top * (dh / 64 * F.STEP * (1 + 2.0 ** -4))
            tol = (F.BF16 + F.STEP * (1 + 2.0 ** -4) + 2 * ds) * mag + 1e-6
            tol = tol + F.BF16 * (np.abs(want) + tol)
            g = got[cu[b] + r]
            assert (np.abs(g - want[0]) <= tol[0]).all(), (b, r)
            if hi - lo > 1:
                assert np.linalg.norm(g - want[0]) <= 2.0 ** -7 * np.linalg.norm(want[0]), (b, r)


@pytest.mark.parametrize("dh", [64, 128, 256])
@pytest.mark.parametrize("nq,window", [(1, 0), (5, 0), (16, 300)])
def test_attention_over_a_cache_said_to_be_large(gpu_ctx, dh, nq, window):
    """Few columns over more pages than the memory's cache holds, by what max_len says, read
    past the L2: the results of the same pages read through it, but for the ranges' joins."""
    rng = np.random.default_rng(dh + nq)
    past, fresh = [700, 64, 0, 1300], [nq, 1, nq, nq]
    pages, table, cu, blk, lens, slots = F.batch_of(rng, past, fresh)
    c = O.Cache(pages, 2, dh)
    acu = np.concatenate([[0], np.cumsum(lens)]).astype(I32)
    asl = np.concatenate([table[b, np.arange(n) // 64].astype(np.int64) * 64 + np.arange(n) % 64
                          for b, n in enumerate(lens)])
    k, v = rng.standard_normal((2, len(asl), 2, dh))
    c.append(k, v, acu, asl)
    q = rng.standard_normal((int(cu[-1]), 4, dh))
    for max_len in (int(max(lens)), 3_000_000):
        for dtype, out_bf16 in (("bf16", True), ("f32", False)):
            got, val = F.attend(gpu_ctx, c, q, dtype, table, cu, lens, dh ** -0.5, True, window,
                                out_bf16, max_len=max_len)
            F.check_attention(c, got, val, table, cu, lens, dh ** -0.5, True, window, dtype, out_bf16)


@pytest.mark.parametrize("dh,kv,nq", [(64, 16, 300), (128, 8, 300), (256, 2, 300)])
def test_wide_attention_of_scores_far_apart(gpu_ctx, dh, kv, nq):
    """Blocks whose scores lie up to 896 apart, in the form of four tiles per workgroup."""
    rng = np.random.default_rng(dh)
    steps = [240, 0, 60, 288, 448, -448, 448, 0]
    batch = {64: 6, 128: 12, 256: 30}[dh]
    n = 64 * len(steps) + 37
    pages, table, cu, blk, lens, slots = F.batch_of(rng, [n - nq] * batch, [nq] * batch)
    c = O.Cache(pages, kv, dh)
    k = np.zeros((batch * n, kv, dh))
    k[:, :, 1] = np.tile(np.resize(np.repeat(steps, 64), n), batch)[:, None]
    k[:, :, dh - 3] = rng.integers(0, 5, (batch * n, kv)) / 4
    v = rng.standard_normal((batch * n, kv, dh))
    asl = np.concatenate([table[b, np.arange(n) // 64].astype(np.int64) * 64 + np.arange(n) % 64
                          for b in range(batch)])
    c.append(k, v, np.arange(batch + 1) * n, asl)
    q = np.zeros((batch * nq, 2 * kv, dh))
    q[:, :, 1] = q[:, :, dh - 3] = 1.0
    got, val = F.attend(gpu_ctx, c, q, "bf16", table, cu, lens, 1.0, True, 0, False)
    for b in (0, batch - 1):
        kk, vv = c.rows(table[b], n)
        for r in (0, 63, 64, 150, nq - 1):
            i = n - nq + r
            want, mag, _ = O.attention(val[cu[b] + r:cu[b] + r + 1], kk[:i + 1], vv[:i + 1], 1.0, False, 0)
            assert (np.abs(got[cu[b] + r] - want[0]) <=
                    (F.BF16 + F.STEP * (1 + 2.0 ** -4)) * mag[0] + 1e-6).all(), (b, r)


@pytest.mark.parametrize("nq", [3, 70])
def test_cache_past_32_bits(gpu_ctx, nq):
    """Pages behind the first 2^31 bytes of a cache, and slots far behind."""
    from rembed_amd import tensor as T
    heads, dh, pages = 4, 256, 40000
    far = np.array([39999, 36000, 1, 33111, 39998], I32)
    rng = np.random.default_rng(nq)
    cache = T.KVCache(gpu_ctx, pages, heads, dh)
    assert cache.k.nbytes > 2 ** 31
    small = O.Cache(5, heads, dh)
    n = 5 * 64 - 9
    k, v = rng.standard_normal((2, n, heads, dh))
    k, v = F.bf16(k)[0].astype(np.float64), F.bf16(v)[0].astype(np.float64)
    cu, blk, lens, slots, pos, _ = O.plan([0], [n], far, np.zeros((1, 5), I32), n)
    F.append(gpu_ctx, cache, k, v, "bf16", cu, blk, slots)
    small.append(k, v, cu, np.arange(n, dtype=np.int64))
    q = rng.standard_normal((nq, 8, dh))
    qcu = np.array([0, nq], I32)
    got, val = F.attend(gpu_ctx, cache_view(cache), q, "bf16", far[None], qcu, lens, dh ** -0.5, True,
                        0, True)
    F.check_attention(small, got, val, np.arange(5)[None], qcu, lens, dh ** -0.5, True, 0, "bf16", True)


def cache_view(cache):
    """What attend takes in place of an oracle's cache."""
    cache.heads = cache.kv_heads
    return cache


@pytest.mark.parametrize("nq,past", [(1, 300), (20, 300), (300, 70)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_of_the_longest_windows(gpu_ctx, nq, past, causal):
    """A window of 2^31 - 1 is none, also for queries that lie before every key."""
    rng = np.random.default_rng(nq)
    pages, table, cu, blk, lens, slots = F.batch_of(rng, [past, 0], [nq, 40])
    c = O.Cache(pages, 2, 64)
    acu = np.concatenate([[0], np.cumsum(lens)]).astype(I32)
    asl = np.concatenate([table[b, np.arange(n) // 64].astype(np.int64) * 64 + np.arange(n) % 64
                          for b, n in enumerate(lens)])
    k, v = rng.standard_normal((2, len(asl), 2, 64))
    c.append(k, v, acu, asl)
    qcu = np.array([0, nq, nq + 90], I32)  # 50 queries of the second before its keys
    q = rng.standard_normal((nq + 90, 4, 64))
    for window in (2 ** 31 - 1, 2 ** 31 - 60, 2 ** 30):
        got, val = F.attend(gpu_ctx, c, q, "bf16", table, qcu, lens, 0.125, causal, window, True)
        F.check_attention(c, got, val, table, qcu, lens, 0.125, causal, 0, "bf16", True)
        if causal:
            assert (got[nq:nq + 50] == 0).all()


class Part:
    """Elements of a device buffer from `first` on."""

    def __init__(self, ctx, ptr, size):
        self.ctx, self.ptr, self.size = ctx, ptr, size

    def read(self, first, dtype, n):
        from rembed_amd import _lib
        out = np.empty(n, dtype)
        _lib.check(_lib.lib.rh_memcpy_d2h(self.ctx.h, out.ctypes.data,
                                          self.ptr + first * out.itemsize, out.nbytes))
        return out


@pytest.mark.parametrize("fits", [True, False])
def test_plan_of_the_most_rows(gpu_ctx, fits):
    """2^31 - 1 rows, whose last loops pass 2^31; one text of most of them, or too long for its
    table."""
    from rembed_amd import tensor as T
    ctx, rows = gpu_ctx, 2 ** 31 - 1
    n = [70, 2 ** 31 - 300, 100]
    blocks = -(-n[1] // 64)
    need = 2 + blocks + 2
    free = np.arange(5, need + 5, dtype=I32)
    ldt = blocks if fits else blocks - 1
    table = ctx.alloc(3 * ldt * 4)
    slots, pos = ctx.alloc(rows * 8), ctx.alloc(rows * 4)
    cu, blk, lens, status = (ctx.alloc(x) for x in (16, 16, 12, 16))
    T.CachePlan(ctx, ctx.upload(np.zeros(3, I32)), ctx.upload(np.array(n, I32)), 3, ctx.upload(free),
                need, table, ldt, cu, blk, lens, slots, pos, rows, status)
    ctx.sync()
    S, P = Part(ctx, slots.ptr, rows), Part(ctx, pos.ptr, rows)
    got = status.download(I32, (4,)).tolist()
    if not fits:
        assert got == [2, 0, 0, 0]
        for at in (0, 2 ** 30, rows - 5000):
            assert (S.read(at, np.int64, 5000) == -1).all() and (P.read(at, I32, 5000) == 0).all()
        return
    total = sum(n)
    assert got == [0, total, need, need] and cu.download(I32, (4,)).tolist() == [0, 70, n[1] + 70, total]
    for at in (70, 2 ** 30 + 1, total - 100 - 5000):
        i = np.arange(at - 70, at - 70 + 5000, dtype=np.int64)
        assert np.array_equal(P.read(at, I32, 5000), i)
        assert np.array_equal(S.read(at, np.int64, 5000), (2 + i // 64 + 5) * 64 + i % 64)
    i = np.arange(100)
    assert np.array_equal(S.read(total - 100, np.int64, 100), (2 + blocks + i // 64 + 5) * 64 + i % 64)
    tail = rows - total
    assert (S.read(total, np.int64, tail) == -1).all() and (P.read(total, I32, tail) == 0).all()
