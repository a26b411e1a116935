"""Performance cases of the 8-bit floating-point operators, through the public entry points.

Decoder embedders put an instruction before every query. Its keys and values
are the same for all of them, so a server holds them in a paged cache and runs
only what is new. The operators are what such a forward calls per layer:

* kind "plan": block tables, slot map and row offsets of a batch, built on the
  GPU from the requests' lengths (tensor.CachePlan);
* kind "append": new K and V rows into the cache, held as e4m3 with one
  exponent for each block of 64 tokens and head (tensor.CacheAppend);
* kind "attend": causal or full attention of the new rows over that cache
  (tensor.CacheAttention);
* kind "linear": one dense layer on e4m3 weights with an exponent for each
  128 x 128 block; fp32 or bf16 rows become e4m3 with an exponent for each 128
  values of a row, bf16 rows come out (tensor.LinearFP8).

A scale is 2^(x - 127) for a byte x: the smallest with which the block's
largest value is at most 448. It is exact, so the 8-bit values are their
type's nearest.
"""
import math
import random

import torch

own = False

BLOCK = 64
ACT = {"none": 0, "gelu": 1, "swiglu": 2}


def _plan(name, batch, past_lo, past_hi, fresh_lo, fresh_hi):
    return {"name": name, "kind": "plan", "batch": batch, "past_lo": past_lo, "past_hi": past_hi,
            "fresh_lo": fresh_lo, "fresh_hi": fresh_hi}


def _append(name, batch, kv_heads, dh, dtype, past_lo, past_hi, fresh_lo, fresh_hi):
    return {"name": name, "kind": "append", "batch": batch, "kv_heads": kv_heads, "dh": dh,
            "dtype": dtype, "past_lo": past_lo, "past_hi": past_hi, "fresh_lo": fresh_lo,
            "fresh_hi": fresh_hi}


def _attend(name, batch, heads, kv_heads, dh, causal, window, shared, past_lo, past_hi, fresh_lo,
            fresh_hi):
    return {"name": name, "kind": "attend", "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "dh": dh, "causal": causal, "window": window, "shared": shared, "past_lo": past_lo,
            "past_hi": past_hi, "fresh_lo": fresh_lo, "fresh_hi": fresh_hi}


def _linear(name, m, k, n, act, bias, dtype):
    return {"name": name, "kind": "linear", "m": m, "k": k, "n": n, "act": act, "bias": bias,
            "dtype": dtype}


def listed():
    return [
        # One token more for each of 48 running texts: the tables grow by a
        # block now and then. The smallest call; latency counts.
        _plan("plan-token", 48, 1, 8191, 1, 1),
        # A queue of documents, some with a cached beginning, some with
        # nothing new.
        _plan("plan-docs", 512, 0, 512, 0, 700),
        # The token's K and V rows of one layer, into blocks partly filled.
        _append("append-token", 48, 8, 128, "bf16", 1, 1500, 1, 1),
        # Documents behind cached beginnings, whole blocks at a time.
        _append("append-docs", 16, 8, 128, "bf16", 0, 200, 300, 2048),
        # A token for each of 48 texts over a long cache: bound by its bytes.
        _attend("attend-token", 48, 16, 8, 128, True, 0, 0, 500, 8191, 1, 1),
        # Queries behind an instruction of ten blocks that all of them share.
        _attend("attend-query", 32, 16, 8, 128, True, 0, 640, 640, 640, 9, 70),
        # A long document's next 4096 tokens: bound by the matrix cores.
        _attend("attend-chunk", 1, 16, 8, 128, True, 0, 0, 8192, 8192, 4096, 4096),
        # Windowed layers of the 3-head embedder, ragged chunks.
        _attend("attend-window", 4, 3, 1, 256, True, 512, 0, 0, 1000, 300, 2048),
        # One token's q|k|v projection, fp32 rows.
        _linear("linear-token", 1, 1024, 4096, "none", False, "f32"),
        # A few texts' rows through a layer with bias and GELU.
        _linear("linear-rows", 37, 2560, 1024, "gelu", True, "bf16"),
        # A gated MLP's first half on a ragged number of rows, k no multiple
        # of the scales' 128.
        _linear("linear-gated", 1213, 1000, 2560, "swiglu", False, "f32"),
        # Documents through a wide layer.
        _linear("linear-docs", 8192, 4096, 4096, "none", False, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    pick = rng.random()
    if pick < 0.15:
        hi = _log_int(rng, 1, 700)
        batch = _log_int(rng, 1, 512)
        past = _log_int(rng, 1, 8191)
        c = _plan("", batch, rng.choice((0, past // 3)), past, rng.choice((0, 1, hi)), hi)
    elif pick < 0.35:
        hi = _log_int(rng, 1, 2048)
        batch = _log_int(rng, 1, max(1, min(48, 16384 // hi)))
        past = _log_int(rng, 1, 1500)
        c = _append("", batch, rng.choice((1, 2, 3, 8)), rng.choice((64, 128, 256)),
                    rng.choice(("bf16", "f32")), rng.choice((0, past // 2)), past,
                    max(1, int(hi * rng.uniform(0.1, 1.0))), hi)
    elif pick < 0.7:
        dh = rng.choice((64, 128, 256))
        kv = rng.choice((1, 2, 4, 8)) if dh < 256 else rng.choice((1, 2))
        group = rng.choice((1, 2, 3, 4, 8))
        hi = rng.choice((1, _log_int(rng, 1, 2048)))
        # rows of all heads within a quarter of the longest listed chunk's work
        batch = _log_int(rng, 1, max(1, min(48, 16384 // (hi * group))))
        past = _log_int(rng, 1, 8191 if hi * batch < 256 else 2048)
        shared = BLOCK * rng.randint(1, 12) if rng.random() < 0.3 else 0
        c = _attend("", batch, kv * group, kv, dh, rng.random() < 0.8,
                    rng.choice((0, 0, 65, 513)), shared, shared + rng.choice((0, past // 2)),
                    shared + past, max(1, int(hi * rng.uniform(0.1, 1.0))), hi)
    else:
        act = rng.choice(("none", "gelu", "swiglu"))
        m = _log_int(rng, 1, 8192)
        c = _linear("", m, _log_int(rng, 96, 4096), 16 * _log_int(rng, 8, 128), act,
                    act == "gelu" or rng.random() < 0.3, rng.choice(("f32", "bf16")))
        if act == "swiglu":
            c["bias"] = False
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


# ---- inputs ------------------------------------------------------------------------------

def _gen(seed, what=0):
    return torch.Generator(device="cuda").manual_seed(8 * int(seed) + what)


def _lens(case):
    """Past and fresh lengths: part of the case, not of the seed."""
    r = random.Random("%d %d %d" % (case["batch"], case["past_hi"], case["fresh_hi"]))
    past = [r.randint(case["past_lo"], case["past_hi"]) for _ in range(case["batch"])]
    fresh = [r.randint(case["fresh_lo"], case["fresh_hi"]) for _ in range(case["batch"])]
    past[0], fresh[0] = case["past_hi"], case["fresh_hi"]
    return past, fresh


def _blocks_of(n):
    return -(-n // BLOCK)


def _arrays(case, seed):
    """The tables of the batch, as CachePlan gives them: pages in no order."""
    past, fresh = _lens(case)
    shared = case.get("shared", 0) // BLOCK
    need = [_blocks_of(p + f) - shared for p, f in zip(past, fresh)]
    pages = shared + sum(need)
    perm = torch.randperm(pages, generator=_gen(seed, 1), device="cuda").int()
    ldt = shared + max(need)
    table = torch.zeros(len(past), ldt, dtype=torch.int32, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    n = torch.tensor(need, **i32)[:, None]
    first = torch.cumsum(n, 0, dtype=torch.int32) - n + shared
    j = torch.arange(ldt, **i32)[None]
    at = torch.where(j < shared, j, first + j - shared)
    at = torch.where(j < shared + n, at, 0)
    table[:] = perm[at.long()]
    pt, ft = torch.tensor(past, **i32), torch.tensor(fresh, **i32)
    cu = torch.zeros(len(past) + 1, **i32)
    cu[1:] = torch.cumsum(ft, 0)
    touched = torch.where(ft > 0, (pt + ft - 1) // BLOCK - pt // BLOCK + 1, 0)
    blocks = torch.zeros(len(past) + 1, **i32)
    blocks[1:] = torch.cumsum(touched, 0)
    rows = sum(fresh)
    req = torch.repeat_interleave(torch.arange(len(past), device="cuda"), ft.long())
    pos = torch.arange(rows, **i32) - cu[req] + pt[req]
    slots = table[req, (pos // BLOCK).long()].long() * BLOCK + pos % BLOCK
    return {"pages": pages, "table": table, "ldt": ldt, "cu": cu, "blocks": blocks,
            "lens": pt + ft, "slots": slots, "rows": rows, "past": pt, "fresh": ft}


def _values(shape, g, scale=1.0):
    """Normal values, heads and channels of different strength among them."""
    x = torch.randn(shape, generator=g, device="cuda")
    return x * (scale * torch.exp(0.5 * torch.randn(shape[-1], generator=g, device="cuda")))


def _filled(case, seed, pages):
    """A cache whose blocks are all written: bytes and exponents of K and V."""
    h, d = case["kv_heads"], case["dh"]
    got = []
    for what, order in ((2, _k_blocks), (3, _v_blocks)):
        x = _values((pages, h, BLOCK, d), _gen(seed, what))
        e = _exponent(x.abs().amax((2, 3)))
        got += [order(_e4m3(x, e[:, :, None, None])), e.to(torch.uint8)]
    k, ke, v, ve = got
    return {"k": k.view(torch.uint8), "v": v.view(torch.uint8), "k_exp": ke, "v_exp": ve}


_TYPE = {"bf16": torch.bfloat16, "f32": torch.float32}


def _plan_inputs(case, seed):
    r = random.Random(int(seed))
    past = [r.randint(case["past_lo"], case["past_hi"]) for _ in range(case["batch"])]
    fresh = [r.randint(case["fresh_lo"], case["fresh_hi"]) for _ in range(case["batch"])]
    ldt = _blocks_of(case["past_hi"] + case["fresh_hi"])
    held = sum(_blocks_of(p) for p in past)
    n_free = case["batch"] * (_blocks_of(case["fresh_hi"]) + 1)
    pages = torch.randperm(held + n_free, generator=_gen(seed, 1), device="cuda").int()
    table = torch.full((case["batch"], ldt), -1, dtype=torch.int32, device="cuda")
    have = torch.tensor([_blocks_of(p) for p in past], dtype=torch.int32, device="cuda")[:, None]
    j = torch.arange(ldt, dtype=torch.int32, device="cuda")[None]
    at = torch.cumsum(have, 0) - have + j
    table = torch.where(j < have, pages[torch.where(j < have, at, 0)], table)
    i32 = dict(dtype=torch.int32, device="cuda")
    rows = max(1, case["batch"] * case["fresh_hi"])  # a padded batch: some rows stay unused
    return {"past": torch.tensor(past, **i32), "fresh": torch.tensor(fresh, **i32),
            "free": pages[held:].contiguous(), "n_free": n_free, "table": table, "ldt": ldt,
            "rows": rows}


def _linear_inputs(case, seed):
    m, k, n = case["m"], case["k"], case["n"]
    a = _values((m, k), _gen(seed, 1)).to(_TYPE[case["dtype"]])
    g = _gen(seed, 2)
    gates = 2 if case["act"] == "swiglu" else 1
    ws = [torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k) for _ in range(gates)]
    b = torch.randn(n, generator=g, device="cuda") * 0.05 if case["bias"] else None
    return a, ws, b


def _by_blocks(w):
    """w as its e4m3 values stand for, an exponent for each 128 x 128 block."""
    n, k = w.shape
    x = torch.nn.functional.pad(w, (0, -k % 128, 0, -n % 128))
    x = x.view((n + 127) // 128, 128, (k + 127) // 128, 128)
    e = _exponent(x.abs().amax((1, 3), keepdim=True))
    x = _e4m3(x, e).float() * _pow2(e)
    return x.reshape(x.shape[0] * 128, -1)[:n, :k].contiguous()


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


def _inputs(case, seed):
    """What the program holds before the call, on the GPU."""
    kind = case["kind"]
    st = {"case": case}
    if kind == "plan":
        st.update(_plan_inputs(case, seed))
    elif kind == "append":
        st.update(_arrays(case, seed))
        st.update(_filled(case, seed, st["pages"]))
        width = case["kv_heads"] * case["dh"]
        # now and then a token is larger than all its block holds
        x = _values((st["rows"], 2 * width), _gen(seed, 4))
        x[::7] *= 3.0
        st["kv"] = x.to(_TYPE[case["dtype"]])
    elif kind == "attend":
        st.update(_arrays(case, seed))
        st.update(_filled(case, seed, st["pages"]))
        # the fused q|k|v rows of the projection, q first
        q, kv = case["heads"] * case["dh"], case["kv_heads"] * case["dh"]
        st["q"] = torch.randn(st["rows"], q + 2 * kv, generator=_gen(seed, 4),
                              device="cuda").to(torch.bfloat16)
        past, fresh = _lens(case)
        st["max_q"], st["max_len"] = max(fresh), max(p + f for p, f in zip(past, fresh))
    else:
        st["a"], st["ws"], st["b"] = _linear_inputs(case, seed)
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:
        _prepare_own(st)
    elif case["kind"] == "linear":
        st["w"] = [_by_blocks(w) for w in st.pop("ws")]  # the packed weights
    torch.cuda.synchronize()  # the context's stream does not wait for torch's
    return st


# ---- the framework's calls ------------------------------------------------------------

def _prepare_own(st):
    from rembed_amd import _lib
    from rembed_amd import tensor as T
    c, ctx = st["case"], _ctx()
    kind, st["ctx"] = c["kind"], ctx

    def empty(shape, dtype):
        return _Dev(torch.empty(shape, dtype=dtype, device="cuda"))

    if kind == "plan":
        n = c["batch"]
        for name, size, dtype in (("o_cu", n + 1, torch.int32), ("o_blocks", n + 1, torch.int32),
                                  ("o_lens", n, torch.int32), ("o_slots", st["rows"], torch.int64),
                                  ("o_pos", st["rows"], torch.int32),
                                  ("o_status", 4, torch.int32)):
            st[name] = empty(size, dtype)
        for name in ("past", "fresh", "free", "table"):
            st["d_" + name] = _Dev(st[name])
        return
    if kind in ("append", "attend"):
        st["cache"] = T.KVCache(ctx, st["pages"], c["kv_heads"], c["dh"],
                                *[_Dev(st[n]) for n in ("k", "v", "k_exp", "v_exp")])
        for name in ("cu", "blocks", "slots", "table", "lens", "kv" if kind == "append" else "q"):
            st["d_" + name] = _Dev(st[name])
    if kind == "attend":
        st["out"] = empty((st["rows"], c["heads"] * c["dh"]), torch.bfloat16)
        need = T.cache_attention_scratch(c["batch"], st["max_q"], st["max_len"], c["heads"],
                                         c["kv_heads"], c["dh"])
        st["scratch"], st["scratch_bytes"] = empty(max(1, need), torch.uint8), need
    if kind == "linear":
        m, k, n = c["m"], c["k"], c["n"]
        host, b = [w.cpu().numpy() for w in st.pop("ws")], st["b"]
        if c["act"] == "swiglu":
            st["pb"] = T.PackedGated(ctx, _lib.RH_MODE_FP8, host[0], host[1], k, n)
        else:
            st["pb"] = T.PackFP8(ctx, host[0], k, n, None if b is None else b.cpu().numpy())
        st["dst"], st["d_a"] = empty((m, n), torch.bfloat16), _Dev(st["a"])
        st["ldq"] = T.ldq_fp8(k)
        st["qa"] = empty((m, st["ldq"]), torch.uint8)
        st["sa"] = empty(T.fp8_scale_bytes(m, k), torch.uint8)


def _run_own(st):
    from rembed_amd import tensor as T
    c, ctx = st["case"], st["ctx"]
    if c["kind"] == "plan":
        T.CachePlan(ctx, st["d_past"], st["d_fresh"], c["batch"], st["d_free"], st["n_free"],
                    st["d_table"], st["ldt"], st["o_cu"], st["o_blocks"], st["o_lens"],
                    st["o_slots"], st["o_pos"], st["rows"], st["o_status"])
        return {"table": st["table"], **{k[2:]: st[k].tensor for k in
                                         ("o_cu", "o_blocks", "o_lens", "o_slots", "o_pos",
                                          "o_status")}}
    if c["kind"] == "append":
        width = c["kv_heads"] * c["dh"]
        T.CacheAppend(ctx, st["cache"], st["d_kv"], c["dtype"] == "bf16", 2 * width, 0, width,
                      st["d_cu"], st["d_blocks"], st["d_slots"], c["batch"], st["rows"])
        return _cache_out(st)
    if c["kind"] == "attend":
        width = c["heads"] * c["dh"]
        T.CacheAttention(ctx, st["out"], True, width, st["d_q"], True,
                         width + 2 * c["kv_heads"] * c["dh"], 0, st["cache"], st["d_table"],
                         st["ldt"], st["d_cu"], st["d_lens"], c["batch"], st["max_q"],
                         st["max_len"], c["heads"], 1.0 / math.sqrt(c["dh"]), c["causal"],
                         c["window"], st["scratch"], st["scratch_bytes"])
        return st["out"].tensor
    T.LinearFP8(ctx, st["dst"], True, c["n"], st["d_a"], c["dtype"] == "bf16", c["k"], st["pb"],
                c["m"], ACT[c["act"]], st["qa"], st["ldq"], st["sa"])
    return st["dst"].tensor


def _cache_out(st):
    """The cache as its values: e4m3 and their exponents."""
    return {"k": st["k"].view(torch.float8_e4m3fn), "v": st["v"].view(torch.float8_e4m3fn),
            "k_exp": st["k_exp"], "v_exp": st["v_exp"]}


# ---- the plain forms ------------------------------------------------------------------

def _run_plan(st):
    past, fresh, ldt, rows = st["past"], st["fresh"], st["ldt"], st["rows"]
    n = past.shape[0]
    have = (past + BLOCK - 1) // BLOCK
    need = (past + fresh + BLOCK - 1) // BLOCK - have
    first = torch.cumsum(need, 0, dtype=torch.int32) - need
    j = torch.arange(ldt, dtype=torch.int32, device=past.device)[None]
    at = first[:, None] + j - have[:, None]
    new = (j >= have[:, None]) & (j < (have + need)[:, None])
    table = torch.where(new, st["free"][torch.where(new, at, 0).long()], st["table"])
    cu = torch.zeros(n + 1, dtype=torch.int32, device=past.device)
    cu[1:] = torch.cumsum(fresh, 0)
    touched = torch.where(fresh > 0, (past + fresh - 1) // BLOCK - past // BLOCK + 1, 0)
    blocks = torch.zeros_like(cu)
    blocks[1:] = torch.cumsum(touched, 0)
    r = torch.arange(rows, dtype=torch.int32, device=past.device)
    req = (torch.searchsorted(cu, r, right=True) - 1).clamp(max=n - 1)
    used = r < cu[n]
    pos = torch.where(used, past[req] + r - cu[req], 0)
    page = table[req, (pos // BLOCK).long()].long()
    slots = torch.where(used, page * BLOCK + pos % BLOCK, -1)
    zero = torch.zeros((), dtype=torch.int32, device=past.device)
    status = torch.stack([zero, cu[n], need.sum().int(), blocks[n]])
    return {"table": table, "cu": cu, "blocks": blocks, "lens": past + fresh, "slots": slots,
            "pos": pos, "status": status}


def _run_append(st):
    c = st["case"]
    h, d, P = c["kv_heads"], c["dh"], st["pages"]
    x = st["kv"].float().view(st["rows"], 2, h, d)
    # a token's head with a value that is no number is kept as K = NaN, V = 0
    bad = ~torch.isfinite(x).all(-1).all(1)
    x = torch.where(bad[:, None, :, None], 0.0, x)
    page, off = st["slots"] // BLOCK, st["slots"] % BLOCK
    opened = torch.zeros(P, dtype=torch.bool, device=x.device)
    opened[page[off == 0]] = True
    touched = torch.zeros(P, dtype=torch.bool, device=x.device)
    touched[page] = True
    nan = torch.tensor(float("nan"), device=x.device)
    out = {}
    for i, (name, rows_of, blocks_of) in enumerate((("k", _k_rows, _k_blocks),
                                                    ("v", _v_rows, _v_blocks))):
        old = rows_of(st[name], d).view(torch.float8_e4m3fn)
        e_old = st[name + "_exp"].int()
        top = torch.zeros(P, h, device=x.device)
        top.scatter_reduce_(0, page[:, None].expand(-1, h), x[:, i].abs().amax(-1), "amax")
        e = torch.where(opened[:, None], 0, e_old)
        e = torch.where(touched[:, None], torch.maximum(e, _exponent(top)), e)
        kept = torch.where(opened[:, None, None, None], 0.0, old.float())
        down = _pow2(127 - torch.where(opened[:, None], 0, e - e_old).clamp(max=126))
        new = (kept * down[:, :, None, None]).to(torch.float8_e4m3fn)
        rows = _e4m3(x[:, i], e[page][:, :, None])
        if i == 0:
            rows = torch.where(bad[:, :, None], nan, rows.float()).to(torch.float8_e4m3fn)
        new.view(torch.uint8)[page, :, off] = rows.view(torch.uint8)
        out[name] = blocks_of(new.view(torch.uint8)).view(torch.float8_e4m3fn)
        out[name + "_exp"] = e.to(torch.uint8)
    return out


def _run_attend(st):
    c = st["case"]
    heads, h, d, n = c["heads"], c["kv_heads"], c["dh"], c["batch"]
    g, L, nq, rows = heads // h, st["ldt"] * BLOCK, st["max_q"], st["rows"]
    page = st["table"].long()
    kv = []
    for name, rows_of in (("k", _k_rows), ("v", _v_rows)):
        e = _pow2(st[name + "_exp"].int())[page]
        x = rows_of(st[name][page.reshape(-1)], d).view(torch.float8_e4m3fn).float()
        x = x.view(n, st["ldt"], h, BLOCK, d) * e[:, :, :, None, None]
        kv.append(x.transpose(1, 2).reshape(n, h, L, d))
    t = torch.arange(nq, device="cuda")[None]
    count = (st["cu"][1:] - st["cu"][:-1])[:, None]
    row = torch.where(t < count, st["cu"][:-1, None] + t, 0)
    q = st["q"][:, : heads * d].float()[row.long()].view(n, nq, h, g, d)
    q = q.permute(0, 2, 3, 1, 4).reshape(n, h, g * nq, d)
    s = q @ kv[0].transpose(2, 3).contiguous() * (1.0 / math.sqrt(d))
    i = (st["lens"][:, None] - count + t)[:, :, None]
    j = torch.arange(L, device="cuda")[None, None]
    see = (j < st["lens"][:, None, None]) & (t < count)[:, :, None]
    if c["causal"]:
        see = see & (j <= i)
    if c["window"]:
        see = see & ((i - j).abs() < c["window"])
    s = s.view(n, h, g, nq, L).masked_fill(~see[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    v = torch.where((j < st["lens"][:, None, None]).transpose(1, 2)[:, None], kv[1], 0.0)
    o = p.view(n, h, g * nq, L) @ v
    o = o / torch.where(total == 0, 1.0, total).view(n, h, g * nq, 1)
    o = o.view(n, h, g, nq, d).permute(0, 3, 1, 2, 4).reshape(n, nq, heads * d)
    return o[(t < count)].to(torch.bfloat16)


def _run_linear(st):
    c = st["case"]
    m, k = c["m"], c["k"]
    x = torch.nn.functional.pad(st["a"].float(), (0, -k % 128)).view(m, -1, 128)
    e = _exponent(x.abs().amax(2, keepdim=True))
    x = (_e4m3(x, e).float() * _pow2(e)).view(m, -1)[:, :k]
    y = [x @ w.t() for w in st["w"]]
    if c["act"] == "swiglu":
        y = y[0] / (1 + torch.exp(-y[0])) * y[1]
    else:
        y = y[0] if st["b"] is None else y[0] + st["b"]
        if c["act"] == "gelu":
            y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    return y.to(torch.bfloat16)


def run(st):
    if own:
        return _run_own(st)
    return {"plan": _run_plan, "append": _run_append, "attend": _run_attend,
            "linear": _run_linear}[st["case"]["kind"]](st)


# ---- what a pass cannot do without ----------------------------------------------------

def _seen(past, fresh, causal, window):
    """(query, key) pairs of one request."""
    n = past + fresh
    total = 0
    for i in range(past, n):
        hi = i if causal else n - 1
        lo = 0
        if window:
            hi, lo = min(hi, i + window - 1), max(0, i - window + 1)
        total += max(0, hi - lo + 1)
    return total


def work(case):
    kind = case["kind"]
    if kind == "plan":
        n, rows = case["batch"], case["batch"] * case["fresh_hi"]
        return {"bytes": 4 * n * 5 + 12 * rows, "flops": 0}
    if kind == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        each = 4 if case["dtype"] == "f32" else 2
        gates = 2 if case["act"] == "swiglu" else 1
        return {"bytes": m * (each * k + 2 * n) + gates * n * k, "flops": 2 * m * k * n * gates}
    past, fresh = _lens(case)
    h, d = case["kv_heads"], case["dh"]
    if kind == "append":
        each = 4 if case["dtype"] == "f32" else 2
        rows = sum(fresh)
        return {"bytes": 2 * rows * h * d * (each + 1) + 8 * rows, "flops": 0}
    # keys before every query's window are not needed; what is shared counts once
    first = [max(0, p - case["window"] + 1) if case["window"] else 0 for p in past]
    keys = sum(p + f - max(x, case["shared"]) for p, f, x in zip(past, fresh, first))
    keys += max(0, case["shared"] - min(first))
    pairs = sum(_seen(p, f, case["causal"], case["window"]) for p, f in zip(past, fresh))
    return {"bytes": 4 * sum(fresh) * case["heads"] * d + 2 * keys * h * d,
            "flops": 4 * pairs * d * case["heads"]}


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


def _exact_plan(case, seed):
    st = {k: v.tolist() if torch.is_tensor(v) else v
          for k, v in _plan_inputs(case, seed).items()}
    cu, blocks, lens, slots, pos, taken = [0], [0], [], [], [], 0
    for b, (p, f) in enumerate(zip(st["past"], st["fresh"])):
        for j in range(_blocks_of(p), _blocks_of(p + f)):
            st["table"][b][j] = st["free"][taken]
            taken += 1
        at = [st["table"][b][(p + t) // BLOCK] for t in range(f)]
        slots += [at[t] * BLOCK + (p + t) % BLOCK for t in range(f)]
        pos += list(range(p, p + f))
        blocks.append(blocks[-1] + len({(p + t) // BLOCK for t in range(f)}))
        cu.append(cu[-1] + f)
        lens.append(p + f)
    status = [0, cu[-1], taken, blocks[-1]]
    more = st["rows"] - cu[-1]
    return {"table": torch.tensor(st["table"]), "cu": torch.tensor(cu),
            "blocks": torch.tensor(blocks), "lens": torch.tensor(lens),
            "slots": torch.tensor(slots + [-1] * more), "pos": torch.tensor(pos + [0] * more),
            "status": torch.tensor(status)}


def _exact_append(case, seed):
    st = _inputs(case, seed)
    h, d = case["kv_heads"], case["dh"]
    x = st["kv"].double().view(st["rows"], 2, h, d)
    cu, past = st["cu"].tolist(), st["past"].tolist()
    table = st["table"].tolist()
    tok = torch.arange(BLOCK)
    # the places of a block's 64 x dh values in its bytes
    kat = torch.empty(BLOCK, d, dtype=torch.long)
    vat = torch.empty(BLOCK, d, dtype=torch.long)
    col = torch.arange(d)
    kat[:] = ((((col // 64) * 2)[None] + (tok // 32)[:, None]) * 2 + (col % 32 // 16)[None]) * 1024 \
        + ((col % 64 // 32)[None] * 32 + (tok % 32)[:, None]) * 16 + (col % 16)[None]
    vat[:] = ((col // 32 * 2)[None] + (tok // 32)[:, None]) * 1024 \
        + ((tok % 8 // 4)[:, None] * 32 + (col % 32)[None]) * 16 \
        + (tok % 32 // 8 * 4 + tok % 4)[:, None]
    out = {}
    for i, (name, at) in enumerate((("k", kat), ("v", vat))):
        codes = st[name].view(torch.float8_e4m3fn).double()
        exps = st[name + "_exp"].long()
        at = at.cuda()
        for b, p in enumerate(past):
            r = cu[b]
            while r < cu[b + 1]:
                off = (p + r - cu[b]) % BLOCK
                n = min(BLOCK - off, cu[b + 1] - r)
                page = table[b][(p + r - cu[b]) // BLOCK]
                y = x[r:r + n, i]
                s, e = _scale64(y.abs().amax((0, 2)))
                e = e.long() + 127
                blk = codes[page][:, at]
                if off == 0:
                    blk = torch.zeros_like(blk)
                else:
                    e = torch.maximum(e, exps[page])
                    blk = _round64(blk * _two(exps[page] - e)[:, None, None])
                s = _two(e - 127)
                blk[:, off:off + n] = _round64(y.transpose(0, 1) / s[:, None, None])
                codes[page].scatter_(1, at.reshape(1, -1).expand(h, -1), blk.reshape(h, -1))
                exps[page] = e
                r += n
        out[name], out[name + "_exp"] = codes, exps
    return out


def _exact_attend(case, seed):
    st = _inputs(case, seed)
    heads, h, d = case["heads"], case["kv_heads"], case["dh"]
    g = heads // h
    cu, lens, table = st["cu"].tolist(), st["lens"].tolist(), st["table"]
    out = torch.empty(st["rows"], heads * d, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        nq = cu[b + 1] - cu[b]
        at = table[b, : _blocks_of(n)].long()
        for u in range(h):
            two = []
            for name, rows_of in (("k", _k_rows), ("v", _v_rows)):
                x = rows_of(st[name][at, u:u + 1].contiguous(), d).view(torch.float8_e4m3fn)
                e = st[name + "_exp"][at, u].long() - 127
                two.append((x[:, 0].double() * _two(e)[:, None, None]).reshape(-1, d)[:n])
            for a in range(u * g, u * g + g):
                for r in range(0, nq, 2048):  # bounded score rows
                    m = min(2048, nq - r)
                    q = st["q"][cu[b] + r:cu[b] + r + m, a * d:a * d + d].double()
                    s = (q @ two[0].t()) / math.sqrt(d)
                    gap = (torch.arange(r, r + m, device="cuda") + n - nq)[:, None] \
                        - torch.arange(n, device="cuda")[None]
                    if case["causal"]:
                        s = s.masked_fill(gap < 0, -math.inf)
                    if case["window"]:
                        s = s.masked_fill(gap.abs() >= case["window"], -math.inf)
                    out[cu[b] + r:cu[b] + r + m, a * d:a * d + d] = torch.softmax(s, 1) @ two[1]
    return out


def _exact_linear(case, seed):
    a, ws, b = _linear_inputs(case, seed)
    k = case["k"]

    def blocked(x, tall):
        r = x.shape[0]
        y = torch.zeros(-(-r // tall) * tall, -(-k // 128) * 128, dtype=torch.float64,
                        device="cuda")
        y[:r, :k] = x
        y = y.view(y.shape[0] // tall, tall, -1, 128)
        s, _ = _scale64(y.abs().amax((1, 3), keepdim=True))
        return (_round64(y / s) * s).reshape(-1, y.shape[2] * 128)[:r, :k]

    x = blocked(a, 1)
    y = [x @ blocked(w, 128).t() for w in ws]
    if case["act"] == "swiglu":
        return y[0] * torch.sigmoid(y[0]) * y[1]
    y = y[0] if b is None else y[0] + b.double()
    return 0.5 * y * (1 + torch.erf(y / math.sqrt(2.0))) if case["act"] == "gelu" else y


def exact(case, seed):
    return {"plan": _exact_plan, "append": _exact_append, "attend": _exact_attend,
            "linear": _exact_linear}[case["kind"]](case, seed)
