"""Performance cases of the row operators between a decoder layer's products, through the public
entry points.

A layer of a decoder embedder that keeps keys and values in the paged e4m3 cache runs, around its
linears and its attention (perf/operators.py):

* kind "norm": the residual stream takes a block's output in and the next block's rows come out:
  norm of the output, gate, scaled sum, norm of the sum, as rows or as the e4m3 codes and scale
  bytes that the next linear takes (tensor.ResidualNorm);
* kind "rotate": norm of each q and k head, then the rotary turn at the rows' positions
  (tensor.RopeRows): pairs of halves or of neighbours, whole heads or their beginning,
  frequencies as trained or scaled for longer texts;
* kind "append": the same on the way into the cache: q's rows out, K and V as the cache's codes
  (tensor.RopeAppend);
* kind "read": tokens of the cache back as rows of K and V (tensor.CacheRead), to move a cached
  beginning to other positions or off the device.

A scale byte x is 2^(x - 127): the smallest with which the block's largest value is at most 448.
"""
import math
import random

import torch

own = False

BLOCK = 64
HALF, PAIRS = 0, 1                       # layouts of the turn
PLAIN, LINEAR, NTK, YARN, WAVES = range(5)  # how frequencies are scaled
THETA = 1.0e6
_TYPE = {"bf16": torch.bfloat16, "f32": torch.float32}


def _rotate(name, rows, heads, kv_heads, dh, rot, layout, scaling, norm, values, dtype, out):
    return {"name": name, "kind": "rotate", "rows": rows, "heads": heads, "kv_heads": kv_heads,
            "dh": dh, "rot": rot, "layout": layout, "scaling": scaling, "norm": norm,
            "values": values, "dtype": dtype, "out": out}


def _norm(name, m, n, x, y, post, gate, pre, out, codes, scale):
    return {"name": name, "kind": "norm", "m": m, "n": n, "x": x, "y": y, "post": post,
            "gate": gate, "pre": pre, "out": out, "codes": codes, "scale": scale}


def _append(name, batch, heads, kv_heads, dh, rot, layout, scaling, norm, dtype, past_lo, past_hi,
            fresh_lo, fresh_hi):
    return {"name": name, "kind": "append", "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "dh": dh, "rot": rot, "layout": layout, "scaling": scaling, "norm": norm,
            "dtype": dtype, "past_lo": past_lo, "past_hi": past_hi, "fresh_lo": fresh_lo,
            "fresh_hi": fresh_hi}


def _read(name, batch, kv_heads, dh, out, past_hi, fresh_lo, fresh_hi):
    return {"name": name, "kind": "read", "batch": batch, "kv_heads": kv_heads, "dh": dh,
            "out": out, "past_lo": 0, "past_hi": past_hi, "fresh_lo": fresh_lo,
            "fresh_hi": fresh_hi}


def listed():
    return [
        # A token for each of 48 running texts: latency counts.
        _rotate("rotate-token", 48, 16, 8, 128, 128, HALF, PLAIN, True, False, "bf16", "bf16"),
        # Encoder rows, half of a head turns, fp32 rows become attention's bf16 ones.
        _rotate("rotate-part", 1213, 12, 12, 64, 32, PAIRS, LINEAR, False, True, "f32", "bf16"),
        # Documents of a decoder, frequencies scaled for long texts.
        _rotate("rotate-docs", 16384, 16, 8, 128, 128, HALF, YARN, True, False, "bf16", "bf16"),
        # The same 48 tokens between attention's output and the gated MLP's e4m3 rows.
        _norm("norm-token", 48, 1024, "f32", "bf16", "none", "none", "rms", "none", True, 1.0),
        # Norms on both sides of a block, some texts' rows.
        _norm("norm-both", 2111, 768, "f32", "bf16", "rms", "none", "rms", "bf16", False, 1.0),
        # Odd rows of an encoder: fp32, a gate for each row, layer norm with its bias.
        _norm("norm-odd", 1213, 1001, "f32", "f32", "none", "row", "layer", "f32", False, 0.5),
        # Documents through a wide layer: bf16 stream, gate for each channel, e4m3 rows out.
        _norm("norm-docs", 8192, 4096, "bf16", "bf16", "none", "channel", "rms", "none", True, 1.0),
        # One token for each of 48 texts, into blocks partly filled.
        _append("append-token", 48, 16, 8, 128, 128, HALF, PLAIN, True, "bf16", 1, 1500, 1, 1),
        # Windowed embedder's heads from fp32 rows, a quarter of each turns.
        _append("append-part", 5, 3, 1, 256, 64, PAIRS, PLAIN, True, "f32", 0, 1000, 300, 700),
        # Documents behind cached beginnings.
        _append("append-docs", 16, 16, 8, 128, 128, HALF, YARN, True, "bf16", 0, 200, 300, 2048),
        # An instruction of ten blocks, to be cached at other positions.
        _read("read-prefix", 1, 8, 128, "bf16", 0, 640, 640),
        # What 16 texts have in the cache, off the device.
        _read("read-docs", 16, 8, 128, "bf16", 100, 500, 8191),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng, most):
    """Heads, kv heads and head dim whose rows hold at most `most` values of q and k."""
    dh = rng.choice((64, 128, 256))
    kv = rng.choice([h for h in (1, 2, 3, 4, 8) if 2 * h * dh <= most])
    group = rng.choice([g for g in (1, 2, 3, 4, 8) if (g + 1) * kv * dh <= most])
    return kv * group, kv, dh


def draw(rng):
    pick = rng.random()
    scaling = rng.choice((PLAIN, PLAIN, LINEAR, NTK, YARN, WAVES))
    layout, norm = rng.choice((HALF, PAIRS)), rng.random() < 0.5
    if pick < 0.3:
        heads, kv, dh = _heads(rng, 4096)
        if rng.random() < 0.2:  # heads of odd sizes
            dh = 2 * rng.randint(8, dh // 2)
        rot = rng.choice((dh, dh, dh // 4 * 2, 2 * rng.randint(1, dh // 2)))
        c = _rotate("", _log_int(rng, 1, 16384), heads, kv, dh, max(rot, 2), layout,
                    scaling if rot > 2 else PLAIN, norm, rng.random() < 0.3,
                    *rng.choice((("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32"))))
        c["rows"] = max(1, min(c["rows"], (1 << 25) // ((heads + 2 * kv) * dh)))
    elif pick < 0.6:
        m = _log_int(rng, 1, 16384)
        n = _log_int(rng, 64, min(8192, max(64, (1 << 24) // m)))
        if rng.random() < 0.6:
            n = (n + 7) // 8 * 8
        pre = rng.choice(("rms", "rms", "layer"))
        out = rng.choice(("none", "f32", "bf16"))
        c = _norm("", m, n, rng.choice(("f32", "bf16")), rng.choice(("none", "f32", "bf16", "bf16")),
                  rng.choice(("none", "none", "rms", "layer")),
                  rng.choice(("none", "none", "row", "channel")), pre, out,
                  out == "none" or rng.random() < 0.2, rng.choice((1.0, 0.25)))
        if c["y"] == "none":
            c.update(post="none", gate="none", scale=1.0)
    elif pick < 0.85:
        hi = _log_int(rng, 1, 2048)
        batch = _log_int(rng, 1, max(1, min(48, 12288 // hi)))
        past = _log_int(rng, 1, 1500)
        heads, kv, dh = _heads(rng, 4096)
        c = _append("", batch, heads, kv, dh, 16 * rng.choice((dh // 16, dh // 16, dh // 32, 1)),
                    layout, scaling, norm, rng.choice(("bf16", "f32")),
                    rng.choice((0, past // 2)), past, max(1, int(hi * rng.uniform(0.1, 1.0))), hi)
    else:
        hi = _log_int(rng, 1, 8191)
        c = _read("", _log_int(rng, 1, max(1, min(48, 32768 // hi))), rng.choice((1, 2, 3, 8)),
                  rng.choice((64, 128)), rng.choice(("bf16", "f32")),
                  rng.choice((0, _log_int(rng, 1, 300))), max(1, int(hi * rng.uniform(0.1, 1.0))),
                  hi)
    del c["name"]
    return c


# ---- e4m3 with exponents ---------------------------------------------------------------

def _exponent(absmax):
    """The byte x of the smallest 2^(x-127) with absmax <= 448 * 2^(x-127)."""
    bits = absmax.float().view(torch.int32)
    return ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(min=0)


def _pow2(x):
    """2^(x - 127) for the bytes 0..254, as float32."""
    return torch.where(x > 0, x << 23, 0x400000).view(torch.float32)


def _e4m3(x, e):
    """The e4m3 values nearest to x * 2^(127 - e)."""
    return (x.float() * _pow2(254 - e)).to(torch.float8_e4m3fn)


def _k_blocks(x):
    """[pages, heads, 64, dh] -> the cache's order: 1 KiB pieces, each 16 values of 64
    (key, half of a step) pairs; a step is 64 of a key's values."""
    p, h, _, d = x.shape
    x = x.view(p, h, 2, 32, d // 64, 2, 2, 16).permute(0, 1, 4, 2, 6, 5, 3, 7)
    return x.reshape(p, h, BLOCK * d)


def _k_rows(x, d):
    p, h, _ = x.shape
    x = x.view(p, h, d // 64, 2, 2, 2, 32, 16).permute(0, 1, 3, 6, 2, 5, 4, 7)
    return x.reshape(p, h, BLOCK, d)


def _v_blocks(x):
    """[pages, heads, 64, dh] -> the cache's order: 1 KiB pieces, each 16 tokens' values
    of 32 columns, twice: tokens 0..3 of every 8, then 4..7."""
    p, h, _, d = x.shape
    x = x.view(p, h, 2, 4, 2, 4, d // 32, 32).permute(0, 1, 6, 2, 4, 7, 3, 5)
    return x.reshape(p, h, BLOCK * d)


def _v_rows(x, d):
    p, h, _ = x.shape
    x = x.view(p, h, d // 32, 2, 2, 32, 4, 4).permute(0, 1, 3, 6, 4, 7, 2, 5)
    return x.reshape(p, h, BLOCK, d)


def _scale_places(m, n):
    """Where the scale byte of block j of row r lies."""
    r = torch.arange(m, device="cuda")[:, None]
    j = torch.arange((n + 127) // 128, device="cuda")[None]
    return ((j * ((m + 127) // 128) + r // 128) * 32 + r % 32) * 4 + r % 128 // 32


# ---- the turn's frequencies ---------------------------------------------------------------

def _scaled_for(scaling):
    """What a program says of its scaling: factor and length trained at."""
    return {"scaling": scaling, "factor": 1.0 if scaling == PLAIN else 4.0,
            "original": 8192 if scaling in (YARN, WAVES) else 0}


def _frequencies(rot, scaling):
    """Radians a position of each pair (a host list), and what cos and sin are multiplied by."""
    s = _scaled_for(scaling)["factor"]
    theta = THETA * s ** (rot / (rot - 2)) if scaling == NTK else THETA
    plain = [theta ** (-2.0 * i / rot) for i in range(rot // 2)]
    if scaling == LINEAR:
        return [f / s for f in plain], 1.0
    if scaling == YARN:  # pairs that turn over 32 times in 8192 positions stay, under once: / s
        lo, hi = (rot * math.log(8192 / (b * 2 * math.pi)) / (2 * math.log(theta)) for b in (32, 1))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), rot - 1)
        hi = hi + 0.001 if lo == hi else hi
        ramp = [min(max((i - lo) / (hi - lo), 0.0), 1.0) for i in range(rot // 2)]
        return [f / s * r + f * (1 - r) for f, r in zip(plain, ramp)], 0.1 * math.log(s) + 1.0
    if scaling == WAVES:  # the same between 4 times and once in 8192 positions, by wavelength
        smooth = [min(max((8192 * f / (2 * math.pi) - 1) / (4 - 1), 0.0), 1.0) for f in plain]
        return [f / s * (1 - r) + f * r for f, r in zip(plain, smooth)], 1.0
    return plain, 1.0


# ---- inputs ------------------------------------------------------------------------------

def _gen(seed, what=0):
    return torch.Generator(device="cuda").manual_seed(16 * int(seed) + what)


def _lens(case):
    """Past and fresh lengths: part of the case, not of the seed."""
    r = random.Random("%d %d %d" % (case["batch"], case["past_hi"], case["fresh_hi"]))
    past = [r.randint(case["past_lo"], case["past_hi"]) for _ in range(case["batch"])]
    fresh = [r.randint(case["fresh_lo"], case["fresh_hi"]) for _ in range(case["batch"])]
    past[0], fresh[0] = case["past_hi"], case["fresh_hi"]
    return past, fresh


def _arrays(case, seed):
    """The tables of the batch, as CachePlan gives them: pages in no order."""
    past, fresh = _lens(case)
    i32 = dict(dtype=torch.int32, device="cuda")
    pt, ft = torch.tensor(past, **i32), torch.tensor(fresh, **i32)
    need = (pt + ft + BLOCK - 1) // BLOCK
    pages, ldt = int(need.sum()), int(need.max())
    perm = torch.randperm(pages, generator=_gen(seed, 1), device="cuda").int()
    j = torch.arange(ldt, **i32)[None]
    at = (torch.cumsum(need, 0) - need)[:, None] + j
    table = torch.where(j < need[:, None], perm[at.clamp(max=pages - 1).long()], -1)
    cu, blocks = torch.zeros(len(past) + 1, **i32), torch.zeros(len(past) + 1, **i32)
    cu[1:] = torch.cumsum(ft, 0)
    blocks[1:] = torch.cumsum((pt + ft - 1) // BLOCK - pt // BLOCK + 1, 0)
    rows = sum(fresh)
    req = torch.repeat_interleave(torch.arange(len(past), device="cuda"), ft.long())
    pos = torch.arange(rows, **i32) - cu[req] + pt[req]
    slots = table[req, (pos // BLOCK).long()].long() * BLOCK + pos % BLOCK
    return {"pages": pages, "table": table.contiguous(), "ldt": ldt, "cu": cu, "blocks": blocks,
            "slots": slots, "pos": pos, "rows": rows, "past": pt, "fresh": ft}


def _values(shape, g, scale=1.0):
    """Normal values, heads and channels of different strength among them."""
    x = torch.randn(shape, generator=g, device="cuda")
    return x * (scale * torch.exp(0.5 * torch.randn(shape[-1], generator=g, device="cuda")))


def _filled(case, seed, pages):
    """A cache whose blocks are all written: codes and scale bytes of K and V."""
    h, d = case["kv_heads"], case["dh"]
    got = []
    for what, order in ((2, _k_blocks), (3, _v_blocks)):
        x = _values((pages, h, BLOCK, d), _gen(seed, what))
        e = _exponent(x.abs().amax((2, 3)))
        got += [order(_e4m3(x, e[:, :, None, None])), e.to(torch.uint8)]
    k, ke, v, ve = got
    return {"k": k.view(torch.uint8), "v": v.view(torch.uint8), "k_exp": ke, "v_exp": ve}


def _head_norms(case, seed):
    g = _gen(seed, 5)
    if not case["norm"]:
        return None, None
    return tuple(1.0 + 0.3 * torch.randn(case["dh"], generator=g, device="cuda") for _ in "qk")


def _stream_inputs(case, seed):
    m, n, g = case["m"], case["n"], _gen(seed, 6)
    st = {"in": _values((m, n), g, 2.0).to(_TYPE[case["x"]])}
    if case["y"] != "none":
        st["y"] = _values((m, n), g, 0.7).to(_TYPE[case["y"]])
    if case["gate"] != "none":
        st["gate"] = torch.rand((m, n) if case["gate"] == "row" else (n,), generator=g, device="cuda")
    for name in ("post", "pre"):
        if case[name] != "none":
            st[name] = 1.0 + 0.3 * torch.randn(n, generator=g, device="cuda")
            st[name + "_b"] = 0.1 * torch.randn(n, generator=g, device="cuda")
    return st


def _inputs(case, seed):
    """What the program holds before the call, on the GPU."""
    kind = case["kind"]
    st = {"case": case}
    if kind == "norm":
        st.update(_stream_inputs(case, seed))
        return st
    if kind == "rotate":
        st["rows"] = case["rows"]
        # texts behind each other, some of them far into a long one
        start = torch.randint(0, 120000, (1 + case["rows"] // 700,), generator=_gen(seed, 1),
                              device="cuda", dtype=torch.int32)
        t = torch.arange(case["rows"], device="cuda", dtype=torch.int32)
        st["pos"] = start[(t // 700).long()] + t % 700
    else:
        st.update(_arrays(case, seed))
        st.update(_filled(case, seed, st["pages"]))
    if kind != "read":  # the fused q|k|v rows of the projection
        width = (case["heads"] + 2 * case["kv_heads"]) * case["dh"]
        x = _values((st["rows"], width), _gen(seed, 4))
        x[::7] *= 3.0
        st["qkv"] = x.to(_TYPE[case["dtype"]])
        st["q_w"], st["k_w"] = _head_norms(case, seed)
        st["freq"], st["amp"] = _frequencies(case["rot"], case["scaling"])
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:
        _prepare_own(st)
    elif "freq" in st:
        st["freq"] = torch.tensor(st["freq"], dtype=torch.float64, device="cuda")
    torch.cuda.synchronize()  # the context's stream does not wait for torch's
    return st


# ---- the framework's calls ------------------------------------------------------------

class _Dev:
    """A torch tensor where the entry points take a device buffer."""

    def __init__(self, tensor):
        self.tensor, self.ptr = tensor, tensor.data_ptr()


_context = []


def _ctx():
    """The program's one context (one stream), as a server holds it."""
    from rembed_amd import tensor as T
    if not _context:
        _context.append(T.Context(0))
    return _context[0]


def _dev(tensor):
    return None if tensor is None else _Dev(tensor)


def _empty(shape, dtype):
    return _Dev(torch.empty(shape, dtype=dtype, device="cuda"))


def _prepare_own(st):
    """The call as the program holds it: the entry point, its arguments, its outputs."""
    from rembed_amd import tensor as T
    c, ctx = st["case"], _ctx()
    {"norm": _call_norm, "rotate": _call_rotate, "append": _call_append,
     "read": _call_read}[c["kind"]](T, ctx, c, st)


def _call_norm(T, ctx, c, st):
    m, n = c["m"], c["n"]
    w = {k: _dev(st.get(k)) for k in ("post", "pre", "post_b", "pre_b", "gate")}
    norms = [None if c[k] == "none" else T.Norm(w[k], 1e-6) if c[k] == "rms"
             else T.Norm(w[k], 1e-5, w[k + "_b"], layer=True) for k in ("post", "pre")]
    res = T.Residual(*norms, w["gate"], ldg=n if c["gate"] == "row" else 0, y_scale=c["scale"])
    total = _empty((m, n), _TYPE[c["x"]]) if c["y"] != "none" else None
    out = _empty((m, n), _TYPE[c["out"]]) if c["out"] != "none" else None
    codes = scales = None
    if c["codes"]:
        codes = _empty((m, T.ldq_fp8(n)), torch.uint8)
        scales = _Dev(torch.full((T.fp8_scale_bytes(m, n),), 127, dtype=torch.uint8,
                                 device="cuda"))
    st["call"] = T.ResidualNorm
    st["args"] = (ctx, res, _Dev(st["in"]), c["x"] == "bf16", n, _dev(st.get("y")),
                  c["y"] == "bf16", n, total, n, out, c["out"] == "bf16", n, codes,
                  T.ldq_fp8(n), scales, m, n)
    got = {"sum": total, "out": out}
    got = {k: v.tensor for k, v in got.items() if v}
    if codes:
        got.update(codes=codes.tensor.view(torch.float8_e4m3fn),
                   scales=scales.tensor.view(torch.float8_e8m0fnu))
    st["got"] = got


def _rope(T, ctx, c, st):
    """The turn's handle and the norms of q and k heads."""
    norms = [None if w is None else T.Norm(_Dev(w), 1e-6) for w in (st["q_w"], st["k_w"])]
    return T.Rope(ctx, c["rot"], THETA, layout=c["layout"], **_scaled_for(c["scaling"])), norms


def _call_rotate(T, ctx, c, st):
    h, kv, d = c["heads"], c["kv_heads"], c["dh"]
    width = (h + (2 if c["values"] else 1) * kv) * d
    rope, norms = _rope(T, ctx, c, st)
    out = _empty((st["rows"], width), _TYPE[c["out"]])
    st["call"] = T.RopeRows
    st["args"] = (ctx, rope, _Dev(st["qkv"]), c["dtype"] == "bf16", (h + 2 * kv) * d, out,
                  c["out"] == "bf16", width, 0, h * d, (h + kv) * d if c["values"] else -1, h, kv,
                  d, _Dev(st["pos"]), st["rows"], *norms)
    st["got"] = out.tensor


def _cache(T, ctx, c, st):
    return T.KVCache(ctx, st["pages"], c["kv_heads"], c["dh"],
                     *[_Dev(st[n]) for n in ("k", "v", "k_exp", "v_exp")])


def _call_append(T, ctx, c, st):
    h, kv, d = c["heads"], c["kv_heads"], c["dh"]
    rope, norms = _rope(T, ctx, c, st)
    q = _empty((st["rows"], h * d), torch.bfloat16)
    st["call"] = T.RopeAppend
    st["args"] = (ctx, rope, _cache(T, ctx, c, st), _Dev(st["qkv"]), c["dtype"] == "bf16",
                  (h + 2 * kv) * d, 0, h * d, (h + kv) * d, q, True, h * d, h, _Dev(st["pos"]),
                  _Dev(st["cu"]), _Dev(st["blocks"]), _Dev(st["slots"]), c["batch"], st["rows"],
                  *norms)
    # the cache as its values: e4m3 and their powers of two
    st["got"] = {"q": q.tensor, "k": st["k"].view(torch.float8_e4m3fn),
                 "v": st["v"].view(torch.float8_e4m3fn),
                 "k_exp": st["k_exp"].view(torch.float8_e8m0fnu),
                 "v_exp": st["v_exp"].view(torch.float8_e8m0fnu)}


def _call_read(T, ctx, c, st):
    width = 2 * c["kv_heads"] * c["dh"]
    out = _empty((st["rows"], width), _TYPE[c["out"]])
    st["call"] = T.CacheRead
    st["args"] = (ctx, _cache(T, ctx, c, st), _Dev(st["table"]), st["ldt"], _Dev(st["cu"]),
                  _Dev(st["past"]), c["batch"], st["rows"], out, c["out"] == "bf16", width, 0,
                  width // 2)
    st["got"] = out.tensor


# ---- the plain forms ------------------------------------------------------------------

def _normed(x, kind, w, b):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w + b
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w


def _turned(x, st):
    """Heads [rows, h, dh] in 32 bits, turned at the rows' positions."""
    c = st["case"]
    rot = c["rot"]
    angle = st["pos"].double()[:, None] * st["freq"]
    cos, sin = ((f(angle) * st["amp"]).float()[:, None] for f in (torch.cos, torch.sin))
    if c["layout"] == HALF:
        a, b = x[..., : rot // 2], x[..., rot // 2: rot]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((y, x[..., rot:]), -1)


def _split_heads(st):
    """q, k and v heads [rows, h, dh] in 32 bits, q and k normed and turned."""
    c = st["case"]
    h, kv, d = c["heads"], c["kv_heads"], c["dh"]
    x = st["qkv"].float().view(-1, h + 2 * kv, d)
    q, k, v = x[:, :h], x[:, h:h + kv], x[:, h + kv:]
    kind = "rms" if c["norm"] else "none"
    return _turned(_normed(q, kind, st["q_w"], 0), st), _turned(_normed(k, kind, st["k_w"], 0), st), v


def _run_rotate(st):
    q, k, v = _split_heads(st)
    x = torch.cat((q, k, v) if st["case"]["values"] else (q, k), 1)
    return x.flatten(1).to(_TYPE[st["case"]["out"]])


def _run_norm(st):
    c = st["case"]
    m, n = c["m"], c["n"]
    x, got = st["in"].float(), {}
    if c["y"] != "none":
        y = _normed(st["y"].float(), c["post"], st.get("post"), st.get("post_b"))
        x = x + c["scale"] * (y if c["gate"] == "none" else st["gate"] * y)
        got["sum"] = x.to(_TYPE[c["x"]])
    x = _normed(x, c["pre"], st["pre"], st["pre_b"])
    if c["out"] != "none":
        got["out"] = x.to(_TYPE[c["out"]])
    if c["codes"]:
        x = torch.nn.functional.pad(x, (0, -n % 128)).view(m, -1, 128)
        e = _exponent(x.abs().amax(2))
        got["codes"] = _e4m3(x, e[:, :, None]).view(m, -1)
        scales = torch.full((-(-m // 128) * 128 * e.shape[1],), 127, dtype=torch.uint8, device="cuda")
        scales[_scale_places(m, n)] = e.to(torch.uint8)
        got["scales"] = scales.view(torch.float8_e8m0fnu)
    return got


def _run_append(st):
    c = st["case"]
    h, d, P = c["kv_heads"], c["dh"], st["pages"]
    q, k, v = _split_heads(st)
    # a token's head with a value that is no number is kept as K = NaN, V = 0
    bad = ~(torch.isfinite(k).all(-1) & torch.isfinite(v).all(-1))
    page, off = st["slots"] // BLOCK, st["slots"] % BLOCK
    opened = torch.zeros(P, dtype=torch.bool, device=q.device)
    opened[page[off == 0]] = True
    touched = torch.zeros(P, dtype=torch.bool, device=q.device)
    touched[page] = True
    nan = torch.tensor(float("nan"), device=q.device)
    out = {"q": q.flatten(1).to(torch.bfloat16)}
    for name, x, rows_of, blocks_of in (("k", k, _k_rows, _k_blocks), ("v", v, _v_rows, _v_blocks)):
        x = torch.where(bad[:, :, None], 0.0, x)
        old = rows_of(st[name], d).view(torch.float8_e4m3fn)
        e_old = st[name + "_exp"].int()
        top = torch.zeros(P, h, device=x.device)
        top.scatter_reduce_(0, page[:, None].expand(-1, h), x.abs().amax(-1), "amax")
        e = torch.where(opened[:, None], 0, e_old)
        e = torch.where(touched[:, None], torch.maximum(e, _exponent(top)), e)
        kept = torch.where(opened[:, None, None, None], 0.0, old.float())
        down = _pow2(127 - torch.where(opened[:, None], 0, e - e_old).clamp(max=126))
        new = (kept * down[:, :, None, None]).to(torch.float8_e4m3fn)
        rows = _e4m3(x, e[page][:, :, None])
        if name == "k":
            rows = torch.where(bad[:, :, None], nan, rows.float()).to(torch.float8_e4m3fn)
        new.view(torch.uint8)[page, :, off] = rows.view(torch.uint8)
        out[name] = blocks_of(new.view(torch.uint8)).view(torch.float8_e4m3fn)
        out[name + "_exp"] = e.to(torch.uint8).view(torch.float8_e8m0fnu)
    return out


def _run_read(st):
    c = st["case"]
    d = c["dh"]
    r = torch.arange(st["rows"], dtype=torch.int32, device="cuda")
    req = torch.searchsorted(st["cu"], r, right=True) - 1
    pos = r - st["cu"][req] + st["past"][req]
    page, off = st["table"][req, (pos // BLOCK).long()].long(), (pos % BLOCK).long()
    got = []
    for name, rows_of in (("k", _k_rows), ("v", _v_rows)):
        x = rows_of(st[name], d).view(torch.float8_e4m3fn)
        e = _pow2(st[name + "_exp"].int())
        x = x.view(torch.uint8)[page, :, off].view(torch.float8_e4m3fn)
        got.append((x.float() * e[page][:, :, None]).flatten(1))
    return torch.cat(got, 1).to(_TYPE[c["out"]])


def run(st):
    if own:
        st["call"](*st["args"])
        return st["got"]
    return {"rotate": _run_rotate, "norm": _run_norm, "append": _run_append,
            "read": _run_read}[st["case"]["kind"]](st)


# ---- what a pass cannot do without ----------------------------------------------------

_SIZE = {"none": 0, "f32": 4, "bf16": 2}


def work(case):
    kind = case["kind"]
    if kind == "norm":
        m, n = case["m"], case["n"]
        each = _SIZE[case["x"]] * (1 if case["y"] == "none" else 2) + _SIZE[case["y"]]
        each += _SIZE[case["out"]] + (1 if case["codes"] else 0) + (4 if case["gate"] == "row" else 0)
        return {"bytes": m * n * each + 8 * n, "flops": 10 * m * n}
    d, kv = case["dh"], case["kv_heads"]
    if kind == "rotate":
        values = (case["heads"] + (2 if case["values"] else 1) * kv) * d * case["rows"]
        return {"bytes": values * (_SIZE[case["dtype"]] + _SIZE[case["out"]]) + 4 * case["rows"],
                "flops": 8 * values}
    rows = sum(_lens(case)[1])
    if kind == "read":
        return {"bytes": 2 * rows * kv * d * (1 + _SIZE[case["out"]]), "flops": 2 * rows * kv * d}
    each = _SIZE[case["dtype"]]
    return {"bytes": rows * d * (case["heads"] * (each + 2) + 2 * kv * (each + 1)) + 12 * rows,
            "flops": 8 * rows * d * (case["heads"] + kv)}


# ---- the same in 64 bits ----------------------------------------------------------------

def _two(e):
    """2^e in 64 bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _scale64(top):
    """2^e for the least whole e >= -127 with top <= 448 * 2^e, in 64 bits."""
    m, e = torch.frexp(top.double() / 448)
    e = torch.where(m == 0.5, e - 1, e)
    e = torch.where(top == 0, -127, e).clamp(min=-127)
    return _two(e), e


def _round64(x):
    """The e4m3 value nearest to each of |x| <= 448, ties to even, in 64 bits."""
    _, e = torch.frexp(x)
    step = _two((e - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _norm64(x, kind, w, b):
    x = x.double()
    if kind == "layer":
        d = x - x.sum(-1, keepdim=True) / x.shape[-1]
        var = (d ** 2).sum(-1, keepdim=True) / x.shape[-1]
        return d * (var + 1e-5) ** -0.5 * w.double() + b.double()
    if kind == "rms":
        return x * ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) ** -0.5 * w.double()
    return x


def _turn64(x, pos, case):
    """x [rows, h, dh] as complex numbers times e^(i angle)."""
    rot, n = case["rot"], case["rot"] // 2
    freq, amp = _frequencies(rot, case["scaling"])
    angle = pos.double()[:, None] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    by = torch.polar(torch.full_like(angle, amp), angle)[:, None]
    at = torch.arange(n, device=x.device)
    first, second = (at, at + n) if case["layout"] == HALF else (2 * at, 2 * at + 1)
    z = torch.complex(x[..., first], x[..., second]) * by
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _heads64(st):
    c = st["case"]
    h, kv, d = c["heads"], c["kv_heads"], c["dh"]
    x = st["qkv"].double().view(-1, h + 2 * kv, d)
    kind = "rms" if c["norm"] else "none"
    q = _turn64(_norm64(x[:, :h], kind, st["q_w"], None), st["pos"], c)
    k = _turn64(_norm64(x[:, h:h + kv], kind, st["k_w"], None), st["pos"], c)
    return q, k, x[:, h + kv:]


def _exact_rotate(case, seed):
    q, k, v = _heads64(_inputs(case, seed))
    return torch.cat((q, k, v) if case["values"] else (q, k), 1).flatten(1)


def _exact_norm(case, seed):
    st = _inputs(case, seed)
    m, n = case["m"], case["n"]
    x, got = st["in"].double(), {}
    if case["y"] != "none":
        y = _norm64(st["y"], case["post"], st.get("post"), st.get("post_b"))
        gate = st["gate"].double() if "gate" in st else 1.0
        got["sum"] = x = x + gate * y * case["scale"]
    x = _norm64(x, case["pre"], st["pre"], st["pre_b"])
    if case["out"] != "none":
        got["out"] = x
    if case["codes"]:
        y = torch.zeros(m, -(-n // 128) * 128, dtype=torch.float64, device="cuda")
        y[:, :n] = x
        y = y.view(m, -1, 128)
        s, _ = _scale64(y.abs().amax(2))
        got["codes"] = _round64(y / s[:, :, None]).view(m, -1)
        got["scales"] = torch.ones(-(-m // 128) * 128 * s.shape[1], dtype=torch.float64,
                                   device="cuda")
        got["scales"][_scale_places(m, n)] = s
    return got


def _exact_append(case, seed):
    st = _inputs(case, seed)
    h, d = case["kv_heads"], case["dh"]
    q, k, v = _heads64(st)
    cu, past = st["cu"].tolist(), st["past"].tolist()
    table = st["table"].tolist()
    tok, col = torch.arange(BLOCK), torch.arange(d)
    # the places of a block's 64 x dh values in its bytes
    kat = ((((col // 64) * 2)[None] + (tok // 32)[:, None]) * 2 + (col % 32 // 16)[None]) * 1024 \
        + ((col % 64 // 32)[None] * 32 + (tok % 32)[:, None]) * 16 + (col % 16)[None]
    vat = ((col // 32 * 2)[None] + (tok // 32)[:, None]) * 1024 \
        + ((tok % 8 // 4)[:, None] * 32 + (col % 32)[None]) * 16 \
        + (tok % 32 // 8 * 4 + tok % 4)[:, None]
    out = {"q": q.flatten(1)}
    for name, x, at in (("k", k, kat.cuda()), ("v", v, vat.cuda())):
        codes = st[name].view(torch.float8_e4m3fn).double()
        exps = st[name + "_exp"].long()
        for b, p in enumerate(past):
            r = cu[b]
            while r < cu[b + 1]:
                off = (p + r - cu[b]) % BLOCK
                n = min(BLOCK - off, cu[b + 1] - r)
                page = table[b][(p + r - cu[b]) // BLOCK]
                y = x[r:r + n]
                _, e = _scale64(y.abs().amax((0, 2)))
                e = e.long() + 127
                blk = codes[page][:, at]
                if off == 0:
                    blk = torch.zeros_like(blk)
                else:
                    e = torch.maximum(e, exps[page])
                    blk = _round64(blk * _two(exps[page] - e)[:, None, None])
                blk[:, off:off + n] = _round64(y.transpose(0, 1) / _two(e - 127)[:, None, None])
                codes[page].scatter_(1, at.reshape(1, -1).expand(h, -1), blk.reshape(h, -1))
                exps[page] = e
                r += n
        out[name], out[name + "_exp"] = codes, _two(exps - 127)
    return out


def _exact_read(case, seed):
    st = _inputs(case, seed)
    d = case["dh"]
    cu, past, table = st["cu"].tolist(), st["past"].tolist(), st["table"]
    got = []
    for b, p in enumerate(past):
        n = cu[b + 1] - cu[b]
        pages = table[b, : -(-(p + n) // BLOCK)].long()
        two = []
        for name, rows_of in (("k", _k_rows), ("v", _v_rows)):
            x = rows_of(st[name][pages], d).view(torch.float8_e4m3fn).double()
            x = x * _two(st[name + "_exp"][pages].long() - 127)[:, :, None, None]
            two.append(x.transpose(1, 2).reshape(-1, case["kv_heads"] * d)[p:p + n])
        got.append(torch.cat(two, 1))
    return torch.cat(got)


def exact(case, seed):
    return {"rotate": _exact_rotate, "norm": _exact_norm, "append": _exact_append,
            "read": _exact_read}[case["kind"]](case, seed)
