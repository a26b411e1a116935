"""A decoder layer through the public entry points alone: residual norms, e4m3 linears, the rotary
append, attention over the cache. Step after step against numpy in 64 bits, recorded as HIP
graphs, on two contexts at once; a cached beginning moved to other positions; offsets past 32
bits.
"""
import ctypes
import threading

import numpy as np
import pytest

import fp8_oracle as O
import row_oracle as R
import test_fp8_operators as F
import test_fp8_serving as S
import test_row_operators as W

pytestmark = pytest.mark.gpu
I32 = np.int32
KW = dict(theta=1e4, scaling=3, factor=4.0, original=256)


class Layer:
    """One layer with norms on both sides of its blocks, its cache and a step's buffers."""

    def __init__(self, ctx, hidden, heads, kv, dh, inter, batch, pages, ldt, rows, max_len, seed=0):
        from rembed_amd import tensor as T
        rng = np.random.default_rng(seed)
        self.ctx, self.hidden, self.heads, self.kv, self.dh = ctx, hidden, heads, kv, dh
        self.inter, self.batch, self.rows, self.max_len = inter, batch, rows, max_len
        self.width = (heads + 2 * kv) * dh
        weight = lambda n, k: (rng.standard_normal((n, k)) * (1.5 / k ** 0.5)).astype(np.float32)
        self.w = {"qkv": weight(self.width, hidden), "o": weight(hidden, heads * dh),
                  "gate": weight(inter, hidden), "up": weight(inter, hidden),
                  "down": weight(hidden, inter)}
        self.pw = {"qkv": T.PackFP8(ctx, self.w["qkv"], hidden, self.width),
                   "o": T.PackFP8(ctx, self.w["o"], heads * dh, hidden),
                   "mlp": T.PackedGated(ctx, 3, self.w["gate"], self.w["up"], hidden, inter),
                   "down": T.PackFP8(ctx, self.w["down"], inter, hidden)}
        self.val = {n: O.quantize_weight(x.astype(np.float64))[2] for n, x in self.w.items()}
        self.g = {n: rng.uniform(0.5, 1.5, dh if n in "qk" else hidden).astype(np.float32)
                  for n in ("q", "k", "n1", "n2", "n3", "n4", "n5", "scale")}
        dev = {n: ctx.upload(x) for n, x in self.g.items()}
        self.norm = {n: T.Norm(dev[n], 1e-6) for n in self.g}
        # before attention; around it; after the MLP
        self.res = [T.Residual(None, self.norm["n1"]),
                    T.Residual(self.norm["n2"], self.norm["n3"], dev["scale"]),
                    T.Residual(self.norm["n4"], self.norm["n5"], y_scale=0.5)]
        self.rope = T.Rope(ctx, dh, **KW)
        i32 = lambda n: ctx.alloc(n * 4)
        self.past, self.fresh, self.free = i32(batch), i32(batch), i32(pages)
        self.ldt, self.table = ldt, ctx.upload(np.full((batch, ldt), -1, I32))
        self.cu, self.blocks, self.lens, self.status = i32(batch + 1), i32(batch + 1), i32(batch), i32(4)
        self.slots, self.pos = ctx.alloc(rows * 8), i32(rows)
        k = max(hidden, heads * dh, inter)
        self.ldh = T.ldq_fp8(hidden)
        self.qa, self.sa = ctx.alloc(rows * T.ldq_fp8(k)), ctx.alloc(T.fp8_scale_bytes(rows, k))
        self.codes = [ctx.alloc(rows * self.ldh) for _ in "ab"]
        self.scales = [ctx.alloc(T.fp8_scale_bytes(rows, hidden)) for _ in "ab"]
        self.x = ctx.alloc(rows * hidden * 4)
        self.qkv, self.q = ctx.alloc(rows * self.width * 2), ctx.alloc(rows * heads * dh * 2)
        self.att, self.o = ctx.alloc(rows * heads * dh * 2), ctx.alloc(rows * hidden * 2)
        self.x1 = ctx.alloc(rows * hidden * 4)
        self.mid, self.y = ctx.alloc(rows * inter * 2), ctx.alloc(rows * hidden * 4)
        self.out = ctx.alloc(rows * hidden * 4)
        self.oracle = O.Cache(pages, kv, dh, fill=0x55)
        self.cache = F.device_cache(ctx, self.oracle)
        self.need = max(T.cache_attention_scratch(batch, n, max_len, heads, kv, dh)
                        for n in range(1, rows + 1))
        self.scratch = ctx.alloc(self.need)

    def give(self, past, fresh, free, x):
        from rembed_amd import _lib
        for buf, a in ((self.past, np.array(past, I32)), (self.fresh, np.array(fresh, I32)),
                       (self.free, np.array(free, I32)), (self.x, np.ascontiguousarray(x, np.float32))):
            _lib.check(_lib.lib.rh_memcpy_h2d(self.ctx.h, buf.ptr, a.ctypes.data, a.nbytes))

    def step(self, m, n_free, max_q, scratch=None):
        """Enqueues a step of up to m rows."""
        from rembed_amd import tensor as T
        c, h, hd, kd = self.ctx, self.hidden, self.heads * self.dh, self.kv * self.dh
        T.CachePlan(c, self.past, self.fresh, self.batch, self.free, n_free, self.table, self.ldt,
                    self.cu, self.blocks, self.lens, self.slots, self.pos, m, self.status)
        used = W.At(self.status, 4)
        T.ResidualNorm(c, self.res[0], self.x, False, h, None, False, 0, None, 0, None, False, 0,
                       self.codes[0], self.ldh, self.scales[0], m, h, used)
        T.MatMulFP8(c, self.qkv, True, self.width, self.codes[0], self.ldh, self.scales[0],
                    self.pw["qkv"], m)
        T.RopeAppend(c, self.rope, self.cache, self.qkv, True, self.width, 0, hd, hd + kd, self.q, True,
                     hd, self.heads, self.pos, self.cu, self.blocks, self.slots, self.batch, m,
                     self.norm["q"], self.norm["k"])
        T.CacheAttention(c, self.att, True, hd, self.q, True, hd, 0, self.cache, self.table, self.ldt,
                         self.cu, self.lens, self.batch, max_q, self.max_len, self.heads,
                         self.dh ** -0.5, True, 0, scratch or self.scratch, self.need)
        T.LinearFP8(c, self.o, True, h, self.att, True, hd, self.pw["o"], m, 0, self.qa,
                    T.ldq_fp8(hd), self.sa)
        T.ResidualNorm(c, self.res[1], self.x, False, h, self.o, True, h, self.x1, h, None, False, 0,
                       self.codes[1], self.ldh, self.scales[1], m, h, used)
        T.MatMulFP8(c, self.mid, True, self.inter, self.codes[1], self.ldh, self.scales[1],
                    self.pw["mlp"], m, 2)
        T.LinearFP8(c, self.y, False, h, self.mid, True, self.inter, self.pw["down"], m, 0, self.qa,
                    T.ldq_fp8(self.inter), self.sa)
        T.ResidualNorm(c, self.res[2], self.x1, False, h, self.y, False, h, self.x1, h, self.out,
                       False, h, None, 0, None, m, h, used)

    def got(self, m):
        from rembed_amd import tensor as T
        self.ctx.sync()
        bf = lambda b, n: F.from_bf16(b.download(np.uint16, (m, n))).astype(np.float64)
        f = lambda b: b.download(np.float32, (m, self.hidden)).astype(np.float64)
        g = {"qkv": bf(self.qkv, self.width), "q": bf(self.q, self.heads * self.dh),
             "att": bf(self.att, self.heads * self.dh), "o": bf(self.o, self.hidden),
             "mid": bf(self.mid, self.inter), "y": f(self.y), "sum": f(self.x1), "out": f(self.out)}
        for i in (0, 1):
            g["codes%d" % i] = self.codes[i].download(np.uint8, (m, self.ldh))
            raw = self.scales[i].download(np.uint8, (T.fp8_scale_bytes(m, self.hidden),))
            g["scales%d" % i] = O.scale_rows(raw, m, self.ldh // 128)
        return g


def decoded(codes, scales, n):
    return (O.CODES[codes] * np.repeat(O.two(scales.astype(np.int64)), 128, 1))[:, :n]


NONE = (0, None, None, 0)


@pytest.mark.parametrize("heads,kv,dh", [(4, 2, 64), (4, 4, 128), (3, 1, 256)])
def test_layer_steps(gpu_ctx, heads, kv, dh):
    """Every operator's output against 64 bits of what it was given, the cache's bytes after every
    step, and all of it read back."""
    from rembed_amd import tensor as T
    hidden = 192
    L = Layer(gpu_ctx, hidden, heads, kv, dh, 272, 4, 40, 9, 400, 600)
    rng = np.random.default_rng(dh)
    order = rng.permutation(40).astype(I32)
    past, taken = np.zeros(4, int), 0
    table = np.full((4, 9), -1, I32)
    rms = lambda n: (1, L.g[n].astype(np.float64), None, 1e-6)
    for fresh in ([130, 5, 0, 64], [1, 1, 0, 1], [1, 60, 190, 1], [1, 1, 1, 0], [3, 1, 2, 70],
                  [1, 1, 1, 1]):
        m = sum(fresh)
        x = rng.standard_normal((m, hidden)).astype(np.float32)
        free = order[taken:]
        L.give(past, fresh, free, x)
        L.step(m, len(free), max(fresh))
        cu, blocks, lens, slots, pos, status = O.plan(past, fresh, free, table, m)
        g = L.got(m)
        x = x.astype(np.float64)
        _, _, want, far = R.residual(x, None, NONE, rms("n1"), None, 1.0, 1.0)
        W.check_codes({"codes": g["codes0"], "scales": g["scales0"]}, want, far, hidden)
        S.close_linear(g["qkv"], decoded(g["codes0"], g["scales0"], hidden), L.val["qkv"], None, 0, True)
        val = g["qkv"].reshape(m, -1, dh)
        W.check_heads(g["q"].reshape(m, heads, dh), val[:, :heads], heads, 0, dh, dh, 0, KW, pos,
                      [L.g["q"]] * 2, True, (1e-6,) * 2)
        # K as rh_rope_rows turns it in fp32, appended
        turned, read = W.marked(gpu_ctx, m, L.width, False)
        T.RopeRows(gpu_ctx, L.rope, L.qkv, True, L.width, turned, False, L.width, 0, heads * dh, -1, 0,
                   kv, dh, L.pos, m, None, L.norm["k"])
        k = read()[0][:, heads * dh:(heads + kv) * dh].reshape(m, kv, dh).astype(np.float64)
        W.check_heads(k, val[:, heads:heads + kv], kv, 0, dh, dh, 0, KW, pos, [L.g["k"]] * 2, False,
                      (1e-6,) * 2)
        before = [a.copy() for a in (L.oracle.k, L.oracle.k_exp)]
        L.oracle.append(k, val[:, heads + kv:], cu, slots)
        W.same_but_for_norms(L.cache, L.oracle, before)
        F.check_attention(L.oracle, g["att"].reshape(m, heads, dh), g["q"].reshape(m, heads, dh), table,
                          cu, lens, dh ** -0.5, True, 0, "bf16", True)
        S.close_linear(g["o"], g["att"], L.val["o"], None, 0, True)
        x1, _, want, far = R.residual(x, g["o"], rms("n2"), rms("n3"), L.g["scale"].astype(np.float64),
                                      1.0, 1.0)
        W.check_codes({"codes": g["codes1"], "scales": g["scales1"]}, want, far, hidden)
        d = decoded(g["codes1"], g["scales1"], hidden)
        want = F.gated(d @ L.val["gate"].T, d @ L.val["up"].T, 2)
        assert np.linalg.norm(g["mid"] - want) <= (F.BF16 + 3 * F.NORM) * np.linalg.norm(want)
        S.close_linear(g["y"], g["mid"], L.val["down"], None, 0, False)
        # x1 itself has been written over: its fp32 rounding is u of it
        s, so, want, far = R.residual(x1, g["y"], rms("n4"), rms("n5"), None, 1.0, 0.5)
        so = so + 8 * R.U * np.abs(x1).max()
        assert (np.abs(g["sum"] - s) <= R.stored(s, so, False)).all()
        want, far = R.norm(g["sum"], np.zeros_like(s), *rms("n5"), hidden)
        # pre() takes the sum before it is rounded to fp32
        far = far + 2 * R.U * np.abs(want) + R.U * np.abs(want).max()
        assert (np.abs(g["out"] - want) <= R.stored(want, far, False)).all()
        past = past + fresh
        taken += status[2]
    total = int(past.sum())
    cu = np.concatenate([[0], np.cumsum(past)]).astype(I32)
    buf, read = W.marked(gpu_ctx, total, 2 * kv * dh, False)
    T.CacheRead(gpu_ctx, L.cache, L.table, 9, gpu_ctx.upload(cu), None, 4, total, buf, False,
                2 * kv * dh, 0, kv * dh)
    rows, _ = read()
    for b in range(4):
        k, v = L.oracle.rows(table[b], int(past[b]))
        both = np.concatenate([k.reshape(past[b], -1), v.reshape(past[b], -1)], 1)
        assert np.array_equal(rows[cu[b]:cu[b + 1]], both.astype(np.float32))


@pytest.mark.parametrize("fresh,dh", [([1, 1, 1], 128), ([40, 33, 50], 64), ([20, 1, 70], 256)])
def test_recorded_layer_steps(gpu_ctx, fresh, dh):
    """Two layers' steps recorded as graphs, replayed in turn with eager steps and
    synchronizations between, with more rows than the batch uses: the bits of steps launched one
    by one."""
    layers = [Layer(gpu_ctx, 128, 4, 2, dh, 144, 3, 60, 20, 240, 1200, seed=s) for s in (1, 2, 1, 2)]
    rec, eager = layers[:2], layers[2:]
    m, rows = sum(fresh), sum(fresh) + 7
    order = np.random.default_rng(5).permutation(60).astype(I32)
    rng = np.random.default_rng(6)
    past, taken = np.zeros(3, int), 0
    for f in ([70, 64, 3], [1, 66, 61]):
        x = rng.standard_normal((sum(f), 128))
        for a in layers:
            a.give(past, f, order[taken:], x)
            a.step(sum(f), 60 - taken, 80)
            gpu_ctx.sync()
        taken += int(layers[0].status.download(I32, (4,))[2])
        past = past + f
    for a in layers:
        a.give(past, fresh, np.resize(order[taken:], 60), rng.standard_normal((rows, 128)))
    graphs = [S.Recorded(gpu_ctx, lambda a=a: a.step(rows, 60, max(fresh), layers[0].scratch)) for a in rec]
    for turn in range(4):
        x = rng.standard_normal((rows, 128))
        for a in layers:
            a.give(past, fresh, np.resize(order[taken:], 60), x)
        for graph in graphs:
            graph.replay()
        if turn % 2:
            gpu_ctx.sync()
        for a in eager:
            a.step(rows, 60, max(fresh))
        for a, b in zip(rec, eager):
            g, h = a.got(m), b.got(m)
            for name in g:
                assert np.array_equal(g[name], h[name]), (turn, name)
            for name in ("k", "v", "k_exp", "v_exp"):
                n = (getattr(a.cache, name).nbytes,)
                assert np.array_equal(getattr(a.cache, name).download(np.uint8, n),
                                      getattr(b.cache, name).download(np.uint8, n)), (turn, name)
        assert layers[0].status.download(I32, (4,))[0] == 0
        taken += int(layers[0].status.download(I32, (4,))[2])
        past = past + fresh
    for graph in graphs:
        graph.close()


def test_layers_on_two_contexts():
    """Steps on two contexts from two threads: what each gives alone."""
    from rembed_amd import tensor as T

    def work(ctx, seed, out):
        L = Layer(ctx, 256, 8, 2, 128, 272, 4, 60, 20, 600, 1300, seed=seed)
        rng = np.random.default_rng(seed)
        past, taken = np.zeros(4, int), 0
        for fresh in ([150, 90, 3, 200], [1, 1, 1, 1], [1, 140, 1, 1], [1, 1, 1, 1]):
            L.give(past, fresh, np.arange(taken, 60), rng.standard_normal((sum(fresh), 256)))
            L.step(sum(fresh), 60 - taken, max(fresh))
            out.append(L.got(sum(fresh)))
            taken += int(L.status.download(I32, (4,))[2])
            past = past + fresh

    with T.Context(0) as c1, T.Context(0) as c2:
        alone, both = ([], []), ([], [])
        work(c1, 1, alone[0])
        work(c2, 2, alone[1])
        threads = [threading.Thread(target=work, args=a) for a in ((c1, 1, both[0]), (c2, 2, both[1]))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    for a, b in zip(alone, both):
        assert len(a) == len(b) == 4
        for g, h in zip(a, b):
            for name in g:
                assert np.array_equal(g[name], h[name]), name


@pytest.mark.parametrize("layout,dh,rot", [(0, 128, 128), (1, 64, 32)])
def test_a_beginning_at_other_positions(gpu_ctx, layout, dh, rot):
    """A cached beginning read back, its K turned by the difference, and appended behind another
    text: within the codes' roundings (twice half a step of e4m3, values of a block against its
    largest) of K turned at the new positions."""
    from rembed_amd import tensor as T
    rng = np.random.default_rng(3)
    n, kv, at = 100, 2, 70
    rope = T.Rope(gpu_ctx, rot, layout=layout)
    x, _ = F.bf16(rng.standard_normal((n, 2 * kv * dh)))
    bits = F.bf16(x)[1]
    cache = F.device_cache(gpu_ctx, O.Cache(8, kv, dh))

    def append(img, bf, table, first, n, norope=False):
        free = [p for p in table[0] if p >= 0][-(-first // 64):]
        t = table.copy()
        cu, blk, lens, slots, pos, _ = O.plan([first], [n], free, t, n)
        up = gpu_ctx.upload
        if norope:
            T.CacheAppend(gpu_ctx, cache, img, bf, 2 * kv * dh, 0, kv * dh, up(cu), up(blk), up(slots), 1, n)
        else:
            T.RopeAppend(gpu_ctx, rope, cache, img, bf, 2 * kv * dh, 0, 0, kv * dh, None, False, 0, 0, up(pos),
                         up(cu), up(blk), up(slots), 1, n)
        gpu_ctx.sync()

    old = np.array([[0, 1, -1]], I32)
    new = np.array([[2, 3, 4]], I32)
    before, _ = F.bf16(rng.standard_normal((at, 2 * kv * dh)))
    append(gpu_ctx.upload(F.bf16(before)[1]), True, new, 0, at)  # the other text
    append(gpu_ctx.upload(bits), True, old, 0, n)
    cu = gpu_ctx.upload(np.array([0, n], I32))
    rows = gpu_ctx.alloc(n * 2 * kv * dh * 4)
    T.CacheRead(gpu_ctx, cache, gpu_ctx.upload(old), 3, cu, None, 1, n, rows, False, 2 * kv * dh, 0, kv * dh)
    by = gpu_ctx.upload(np.full(n, at, I32))
    T.RopeRows(gpu_ctx, rope, rows, False, 2 * kv * dh, rows, False, 2 * kv * dh, 0, 0, -1, 0, kv, dh, by, n)
    gpu_ctx.sync()
    append(rows, False, new, at, n, norope=True)
    back = gpu_ctx.alloc(n * 2 * kv * dh * 4)
    T.CacheRead(gpu_ctx, cache, gpu_ctx.upload(new), 3, cu, gpu_ctx.upload(np.array([at], I32)), 1, n, back,
                False, 2 * kv * dh, 0, kv * dh)
    gpu_ctx.sync()
    got = back.download(np.float32, (n, 2, kv, dh)).astype(np.float64)
    val = x.astype(np.float64).reshape(n, 2, kv, dh)
    k, _ = R.turn(val[:, 0], np.zeros((n, kv, dh)), np.arange(n) + at, *R.frequencies(rot), layout == 0)
    # each of two codes is off by half a step: 2^-4 of the value or, under the block's normal
    # numbers, 2^-10 of its power of two (at most twice the block's largest / 448); the first one's
    # errors are turned, so a pair's meet
    top = max(np.abs(val).max(), np.abs(before).max()) * 2 ** 0.5
    each = lambda v: 2.0 ** -4 * np.abs(v) + 2.0 ** -10 * 2 * top / 448
    one, _ = R.turn(val[:, 0], np.zeros((n, kv, dh)), np.arange(n), *R.frequencies(rot), layout == 0)
    _, spread = R.turn(one, each(one), np.full(n, at), *R.frequencies(rot), layout == 0)
    assert (np.abs(got[:, 0] - k) <= spread + each(np.abs(k) + spread)).all()
    v = val[:, 1]
    assert (np.abs(got[:, 1] - v) <= each(v) + each(np.abs(v) + each(v))).all()


# ---- offsets past 32 bits -----------------------------------------------------------------

def put(ctx, ptr, a):
    from rembed_amd import _lib
    a = np.ascontiguousarray(a)
    _lib.check(_lib.lib.rh_memcpy_h2d(ctx.h, ptr, a.ctypes.data, a.nbytes))


def get(ctx, ptr, dtype, shape):
    from rembed_amd import _lib
    a = np.empty(shape, dtype)
    _lib.check(_lib.lib.rh_memcpy_d2h(ctx.h, a.ctypes.data, ptr, a.nbytes))
    return a


def test_rows_past_32_bits(gpu_ctx):
    """Strides of 2^30 values: the third row begins 2^32 bytes and more behind the first."""
    from rembed_amd import tensor as T
    ld, m, rng = 1 << 30, 3, np.random.default_rng(1)
    x, y = gpu_ctx.alloc(m * ld * 2), gpu_ctx.alloc(m * ld * 2)
    small = [rng.standard_normal((m, 512)) for _ in "xy"]
    bits = [F.bf16(a)[1] for a in small]
    for r in range(m):
        for buf, b in ((x, bits[0]), (y, bits[1])):
            put(gpu_ctx, buf.ptr + r * ld * 2, b[r])
    dense = [gpu_ctx.upload(b) for b in bits]
    norm = T.Norm(None, 1e-6)
    res = T.Residual(norm, norm)
    out = gpu_ctx.alloc(m * 512 * 2)
    for n in (512, 509):
        want = gpu_ctx.alloc(m * 512 * 2)
        T.ResidualNorm(gpu_ctx, res, dense[0], True, 512, dense[1], True, 512, None, 0, want, True, 512, None,
                       0, None, m, n)
        T.ResidualNorm(gpu_ctx, res, x, True, ld, y, True, ld, None, 0, out, True, 512, None, 0, None, m, n)
        gpu_ctx.sync()
        assert np.array_equal(out.download(np.uint16, (m, 512))[:, :n], want.download(np.uint16, (m, 512))[:, :n])
    pos = gpu_ctx.upload(np.array([5, 70, 900], I32))
    for dh, rot in ((128, 128), (96, 96), (126, 126)):
        rope = T.Rope(gpu_ctx, rot)
        want = gpu_ctx.alloc(m * 512 * 2)
        T.RopeRows(gpu_ctx, rope, dense[0], True, 512, want, True, 512, 0, 2 * dh, -1, 2, 1, dh, pos, m, norm, norm)
        T.RopeRows(gpu_ctx, rope, x, True, ld, y, True, ld, 0, 2 * dh, -1, 2, 1, dh, pos, m, norm, norm)
        gpu_ctx.sync()
        w = want.download(np.uint16, (m, 512))[:, :3 * dh]
        for r in range(m):
            assert np.array_equal(get(gpu_ctx, y.ptr + r * ld * 2, np.uint16, 3 * dh), w[r])
    # the rotary append from such rows, and its rows read back to such rows
    rope = T.Rope(gpu_ctx, 64)
    cu, blk = gpu_ctx.upload(np.array([0, m], I32)), gpu_ctx.upload(np.array([0, 1], I32))
    slots = gpu_ctx.upload(np.arange(m, dtype=np.int64))
    got = []
    for src, stride in ((dense[0], 512), (x, ld)):
        cache = F.device_cache(gpu_ctx, O.Cache(1, 2, 64))
        q = gpu_ctx.alloc(m * 256 * 2)
        T.RopeAppend(gpu_ctx, rope, cache, src, True, stride, 0, 256, 384, q, True, 256, 4, pos, cu, blk, slots, 1,
                     m, norm, norm)
        table = gpu_ctx.upload(np.zeros((1, 1), I32))
        T.CacheRead(gpu_ctx, cache, table, 1, cu, None, 1, m, y, True, ld, 0, 128)
        gpu_ctx.sync()
        got.append([q.download(np.uint16, (m, 256))] +
                   [getattr(cache, a).download(np.uint8, (getattr(cache, a).nbytes,)) for a in ("k", "v", "k_exp")]
                   + [get(gpu_ctx, y.ptr + r * ld * 2, np.uint16, 256) for r in range(m)])
    for a, b in zip(*got):
        assert np.array_equal(a, b)
    assert got[0][4].any()


def test_rows_of_more_than_a_launch(gpu_ctx):
    """More rows than a launch's threads reach: the last ones are as those of a small call."""
    from rembed_amd import tensor as T
    rng = np.random.default_rng(4)
    norm = T.Norm(None, 1e-6)
    # residual norms: 2^21 rows a launch
    m, n = (1 << 21) + 5, 24
    x = rng.standard_normal((8, n)).astype(np.float32)
    buf, out, want = gpu_ctx.alloc(m * n * 4), gpu_ctx.alloc(m * n * 4), gpu_ctx.alloc(8 * n * 4)
    put(gpu_ctx, buf.ptr + (m - 8) * n * 4, x)
    res = T.Residual(None, norm)
    T.ResidualNorm(gpu_ctx, res, buf, False, n, None, False, 0, None, 0, out, False, n, None, 0, None, m, n)
    T.ResidualNorm(gpu_ctx, res, gpu_ctx.upload(x), False, n, None, False, 0, None, 0, want, False, n, None, 0,
                   None, 8, n)
    gpu_ctx.sync()
    assert np.array_equal(get(gpu_ctx, out.ptr + (m - 8) * n * 4, np.float32, (8, n)),
                          want.download(np.float32, (8, n)))
    # rotary rows, in place: sixteen rows of one head of 32 a workgroup, 2^23 workgroups a launch;
    # and heads of 6, taken value by value, in more steps of a grid than one
    for m, dh in (((1 << 27) + 3, 32), ((1 << 22) + (1 << 20) + 3, 6)):
        x = rng.standard_normal((8, dh)).astype(np.float32)
        bits, pos = F.bf16(x)[1], rng.integers(0, 9999, 8).astype(I32)
        buf, dpos = gpu_ctx.alloc(m * dh * 2), gpu_ctx.alloc(m * 4)
        put(gpu_ctx, buf.ptr + (m - 8) * dh * 2, bits)
        put(gpu_ctx, dpos.ptr + (m - 8) * 4, pos)
        want = gpu_ctx.upload(bits)
        rope = T.Rope(gpu_ctx, dh)
        T.RopeRows(gpu_ctx, rope, buf, True, dh, buf, True, dh, 0, 0, -1, 1, 0, dh, dpos, m, norm)
        T.RopeRows(gpu_ctx, rope, want, True, dh, want, True, dh, 0, 0, -1, 1, 0, dh, gpu_ctx.upload(pos), 8,
                   norm)
        gpu_ctx.sync()
        assert np.array_equal(get(gpu_ctx, buf.ptr + (m - 8) * dh * 2, np.uint16, (8, dh)),
                              want.download(np.uint16, (8, dh)))
        del buf, dpos
