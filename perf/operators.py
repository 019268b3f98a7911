"""The operators of text generation that are timed: what one step of a decoder asks for beside its matrix products.

A case is a dict of plain values; its "op" says which operator it calls.

  plan     block tables and slot maps from the lengths of the requests
  append   new keys and values put into a paged cache
  attend   attention of one new token a request over the paged cache
  select   beam search's choice over beams and vocabulary
  reorder  block tables and half-filled blocks that follow the chosen beams

A cache is two pools (keys, values) of blocks of "bs" tokens.  "order" says how a block lies in
memory: "thd" [token][head][dim], "htd" [head][token][dim].  Lengths and block numbers come from
the case ("mix" seeds the lengths), values from the seed of the state.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
DEV = "cuda"


def listed():
    return [
        # a decode step of four requests: what a call costs
        dict(name="plan_decode_4", op="plan", requests=4, bs=16, max_blocks=64, cached=700, added=1, short=0, mix=1),
        # prompts of many requests at once, blocks and slot map nearly used up: the last requests do not fit any more
        dict(name="plan_prompts_2000", op="plan", requests=2000, bs=16, max_blocks=512, cached=300, added=1500, short=1, mix=2),
        # one step of 32 requests in half precision
        dict(name="append_decode_32", op="append", tokens=32, kv=8, dim=128, bs=16, blocks=4096, order="thd", type="bf16", cache="bf16", skip=0),
        # a prompt of an odd length, projections in 32 bits, a cache in 16, heads in front of tokens; the encoder's head sizes
        dict(name="append_prompt_8191", op="append", tokens=8191, kv=12, dim=64, bs=32, blocks=1024, order="htd", type="f32", cache="f16", skip=1),
        # a single request at the encoder's sizes (12 heads of 64, 32 bits) and its length: latency
        dict(name="attend_1x384_f32", op="attend", requests=1, kv=12, group=1, dim=64, bs=16, order="thd", type="f32", cache="f32",
             longest=384, spread=0, window=0, empty=0, mix=3),
        # a batch in service, requests of every age, grouped heads
        dict(name="attend_64xmixed_bf16", op="attend", requests=64, kv=8, group=4, dim=128, bs=16, order="thd", type="bf16", cache="bf16",
             longest=8192, spread=1, window=0, empty=1, mix=4),
        # few requests with very long caches
        dict(name="attend_3x131071_f16", op="attend", requests=3, kv=8, group=8, dim=128, bs=64, order="htd", type="f16", cache="f16",
             longest=131071, spread=0, window=0, empty=0, mix=5),
        # activations in 32 bits over a 16-bit cache, odd block size, head size 80, a sliding window
        dict(name="attend_17xwindow_f32_bf16", op="attend", requests=17, kv=5, group=3, dim=80, bs=24, order="thd", type="f32", cache="bf16",
             longest=6000, spread=1, window=1000, empty=1, mix=6),
        # one request, four beams, the encoder's vocabulary, an odd row length
        dict(name="select_1x4_f32", op="select", requests=1, beams=4, vocab=30522, select=8, type="f32", ended=0),
        # a batch of beams over a large odd vocabulary in half precision
        dict(name="select_48x8_bf16", op="select", requests=48, beams=8, vocab=128257, select=16, type="bf16", ended=1),
        # one request's beams
        dict(name="reorder_4", op="reorder", rows=4, layers=6, kv=12, dim=64, bs=16, order="thd", cache="f32", longest=384, mix=11),
        # a batch of beams through all layers of a larger model
        dict(name="reorder_256", op="reorder", rows=256, layers=24, kv=8, dim=128, bs=16, order="htd", cache="bf16", longest=1500, mix=8),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("plan", "append", "append", "attend", "attend", "attend", "attend", "select", "select", "reorder"))
    mix = rng.randrange(1, 1 << 20)
    bs = rng.choice((8, 16, 16, 24, 32, 64, 128))
    dim = rng.choice((32, 40, 64, 64, 72, 80, 96, 128, 128, 128, 192, 256))
    order = rng.choice(("thd", "htd"))
    pair = rng.choice((("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "bf16")))
    if op == "plan":
        return dict(op=op, requests=_log_int(rng, 1, 4000), bs=bs, max_blocks=_log_int(rng, 16, 1024), cached=_log_int(rng, 1, 2000),
                    added=rng.choice((1, 1, _log_int(rng, 2, 1000))), short=rng.choice((0, 1)), mix=mix)
    if op == "append":
        return dict(op=op, tokens=_log_int(rng, 1, 16000), kv=rng.choice((1, 2, 4, 5, 8, 12)), dim=dim, bs=bs, blocks=-(-20000 // bs),
                    order=order, type=pair[0], cache=pair[1], skip=rng.choice((0, 1)))
    if op == "select":
        while True:
            c = dict(op=op, requests=_log_int(rng, 1, 64), beams=rng.choice((1, 2, 3, 4, 5, 8, 16)), vocab=_log_int(rng, 300, 152000),
                     select=rng.choice((1, 2, 5, 8, 16, 32)), type=pair[0], ended=rng.choice((0, 1)))
            if c["requests"] * c["beams"] * c["vocab"] < 3e7:
                return c
    while op == "reorder":
        c = dict(op=op, rows=_log_int(rng, 1, 200), layers=rng.choice((1, 6, 12, 24)), kv=rng.choice((1, 2, 4, 8, 12)), dim=dim,
                 bs=rng.choice((8, 16, 24, 32)), order=order, cache=pair[1], longest=_log_int(rng, 8, 1500), mix=mix)
        if (c["rows"] + 64) * c["layers"] * c["kv"] * dim * c["bs"] < 3e8:
            return c
    while True:
        c = dict(op=op, requests=_log_int(rng, 1, 100), kv=rng.choice((1, 2, 4, 5, 8, 12)), group=rng.choice((1, 1, 2, 3, 4, 7, 8, 16, 20)),
                 dim=dim, bs=bs, order=order, type=pair[0], cache=pair[1], longest=_log_int(rng, 1, 60000), spread=rng.choice((0, 1, 1)),
                 window=rng.choice((0, 0, 0, _log_int(rng, 1, 4000))), empty=rng.choice((0, 1)), mix=mix)
        if c["requests"] * c["longest"] * c["kv"] * dim < 2.5e8 and c["requests"] * c["longest"] * c["kv"] * c["group"] < 1e8:
            return c


# ---- what a case says about lengths ------------------------------------------------------------
def _lengths(c):
    """The cached tokens of each request: all of "longest", or spread below it over the logarithm; one empty where the case asks for it."""
    r = random.Random(c["mix"])
    n = c["requests"]
    v = [_log_int(r, 1, c["longest"]) if c["spread"] else c["longest"] for _ in range(n)]
    v[r.randrange(n)] = c["longest"]
    if c["empty"] and n > 1:
        v[(v.index(c["longest"]) + 1) % n] = 0
    return v


def _seen(c):
    return [min(n, c["window"]) if c["window"] else n for n in _lengths(c)]


def _plan_lengths(c):
    """(cached, added) of each request."""
    r = random.Random(c["mix"])
    room = c["max_blocks"] * c["bs"]
    cached = [min(room - 1, _log_int(r, 1, 2 * c["cached"]) - 1) for _ in range(c["requests"])]
    added = [c["added"] if c["added"] == 1 else _log_int(r, 1, 2 * c["added"]) for _ in cached]
    return cached, added


def _plan_room(c):
    """(entries of the free list, entries of the slot map): enough, or too few for the last requests."""
    cached, added = _plan_lengths(c)
    bs = c["bs"]
    need = sum(-(-(a + b) // bs) - -(-a // bs) for a, b in zip(cached, added))
    return (max(1, need * 7 // 8), max(1, sum(added) * 15 // 16)) if c["short"] else (need + 16, sum(added) + 8)


def _fill(c):
    """Tokens of each beam's cache."""
    r = random.Random(c["mix"])
    return [_log_int(r, 1, c["longest"]) for _ in range(c["rows"])]


def work(c):
    op = c["op"]
    if op == "plan":
        cached, added = _plan_lengths(c)
        bs = c["bs"]
        need = sum(-(-(a + b) // bs) - -(-a // bs) for a, b in zip(cached, added))
        slots = _plan_room(c)[1]
        return {"bytes": 4 * (4 * c["requests"] + 2 * need + slots), "flops": 0}
    if op == "append":
        return {"bytes": c["tokens"] * (4 + 2 * c["kv"] * c["dim"] * (BYTES[c["type"]] + BYTES[c["cache"]])), "flops": 0}
    if op == "attend":
        seen, heads = sum(_seen(c)), c["kv"] * c["group"]
        return {"bytes": 2 * seen * c["kv"] * c["dim"] * BYTES[c["cache"]] + c["requests"] * heads * (2 * c["dim"] * BYTES[c["type"]] + 4)
                + 4 * sum(-(-n // c["bs"]) for n in _seen(c)), "flops": 4 * seen * heads * c["dim"]}
    if op == "select":
        n = c["requests"] * c["beams"] * c["vocab"]
        return {"bytes": n * BYTES[c["type"]] + 12 * c["requests"] * c["select"], "flops": 4 * n}
    fill, moved = _fill(c), 0
    for i, p in enumerate(_parents(c)):
        if p != i:
            moved += fill[p] % c["bs"]
    return {"bytes": 4 * moved * c["layers"] * c["kv"] * c["dim"] * BYTES[c["cache"]] + 8 * sum(-(-n // c["bs"]) for n in fill) + 20 * c["rows"], "flops": 0}


def _parents(c):
    """Beams of four (or the rest) choose among themselves; about a third stay where they are."""
    r = random.Random(c["mix"] + 1)
    return [i if r.random() < 0.3 else min(c["rows"] - 1, i // 4 * 4 + r.randrange(4)) for i in range(c["rows"])]


# ---- what a program holds ----------------------------------------------------------------------
def _ints(v, kind=torch.int32):
    return torch.tensor(v, dtype=kind).to(DEV)


def _normal(shape, kind, gen):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32 if kind == "f32" else DTYPES[kind])


def _pools(c, blocks, gen, layers=None):
    """Key and value pools as they lie in memory, and the [..., block, token, head, dim] views of them."""
    shape = (blocks, c["bs"], c["kv"], c["dim"]) if c["order"] == "thd" else (blocks, c["kv"], c["bs"], c["dim"])
    shape = shape if layers is None else (layers,) + shape
    pools = [_normal(shape, c["cache"], gen) for _ in range(2)]
    return pools, [p if c["order"] == "thd" else p.transpose(-3, -2) for p in pools]


def prepare(c, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    cpu = np.random.default_rng(seed)
    st = {"c": c}
    op = c["op"]
    if op == "plan":
        cached, added = _plan_lengths(c)
        free, room = _plan_room(c)
        bs, rows = c["bs"], c["requests"]
        have = [-(-n // bs) for n in cached]
        order = cpu.permutation(sum(have) + free).astype(np.int32)
        table = np.full((rows, c["max_blocks"]), -1, np.int32)
        table[np.arange(c["max_blocks"])[None, :] < np.asarray(have)[:, None]] = order[:sum(have)]
        st.update(cached=_ints(cached), added=_ints(added), free=torch.from_numpy(order[sum(have):].copy()).to(DEV), blocks=len(order),
                  table=torch.from_numpy(table).to(DEV), lengths=_ints([0] * rows), starts=_ints([0] * (rows + 1)), slots=_ints([0] * room),
                  counts=_ints([0, 0, 0]))
    elif op == "append":
        st["pools"], st["views"] = _pools(c, c["blocks"], gen)
        # rows of one projection: keys, then values
        st["kv_rows"] = _normal((c["tokens"], 2, c["kv"], c["dim"]), c["type"], gen)
        slots = cpu.permutation(c["blocks"] * c["bs"])[:c["tokens"]].astype(np.int32)
        if c["skip"]:
            slots[cpu.random(c["tokens"]) < 0.05] = -1
        st["slots"] = torch.from_numpy(slots).to(DEV)
    elif op == "attend":
        lengths = _lengths(c)
        have = [-(-n // c["bs"]) for n in lengths]
        width = max(1, max(have))
        order = cpu.permutation(sum(have) + 3).astype(np.int32)
        table = np.full((c["requests"], width), -1, np.int32)
        table[np.arange(width)[None, :] < np.asarray(have)[:, None]] = order[:sum(have)]
        st["pools"], st["views"] = _pools(c, len(order), gen)
        heads = c["kv"] * c["group"]
        # the queries' part of a row that holds keys and values behind them
        st["rows"] = _normal((c["requests"], heads + 2 * c["kv"], c["dim"]), c["type"], gen) * 1.5
        st.update(table=torch.from_numpy(table).to(DEV), lengths=_ints(lengths), longest=max(1, max(lengths)),
                  out=torch.zeros((c["requests"], heads, c["dim"]), dtype=DTYPES[c["type"]], device=DEV),
                  lse=torch.zeros((c["requests"], heads), dtype=torch.float32, device=DEV))
    elif op == "select":
        rows = c["requests"] * c["beams"]
        st["logits"] = (_normal((rows, c["vocab"]), "f32", gen) * 2.5).to(DTYPES[c["type"]])
        st["scores"] = -torch.rand((rows,), generator=gen, device=DEV) * 8
        st["ended"] = (torch.rand((rows,), generator=gen, device=DEV) < 0.1).to(torch.uint8) if c["ended"] else None
        pick = (c["requests"], c["select"])
        st.update(best=torch.zeros(pick, device=DEV), parents=torch.zeros(pick, dtype=torch.int32, device=DEV), tokens=torch.zeros(pick, dtype=torch.int32, device=DEV))
    else:
        fill = _fill(c)
        width = -(-c["longest"] // c["bs"]) + 1
        used = max(64, 2 * c["rows"])
        order = cpu.permutation(used + c["rows"]).astype(np.int32)
        st["pools"], st["views"] = _pools(c, len(order), gen, c["layers"])
        st.update(fill=_ints(fill), parents=_ints(_parents(c)), spare=torch.from_numpy(order[used:].copy()).to(DEV),
                  table=torch.from_numpy(order[cpu.integers(0, used, (c["rows"], width))]).to(DEV),
                  table_out=torch.full((c["rows"], width), -1, dtype=torch.int32, device=DEV), lengths_out=_ints([0] * c["rows"]))
    if op in ("append", "attend", "reorder"):
        v = st["views"][0]
        st["strides"] = (v.stride(-4), v.stride(-3), v.stride(-2))
    return st


def run(st):
    op = st["c"]["op"]
    if own:
        return {"plan": _own_plan, "append": _own_append, "attend": _own_attend, "select": _own_select, "reorder": _own_reorder}[op](st)
    return {"plan": _plan, "append": _append, "attend": _attend, "select": _select, "reorder": _reorder}[op](st)


# ---- the framework's operators -----------------------------------------------------------------
def _kept(st, make):
    """What a program sets up once for its cache: descriptors, and a workspace where the operator wants one."""
    if "desc" not in st:
        from reef_amd import binding
        st["B"] = binding
        st["desc"] = make(binding)
    return st["B"], st["desc"]


def _must(B, status):
    if status != 0:
        raise RuntimeError(B.last_error())


def _layout(B, st):
    c = st["c"]
    return B.CacheLayout(B.TYPES[c["cache"]], st["views"][0].shape[-4], c["bs"], c["kv"], c["dim"], *st["strides"])


def _own_plan(st):
    c = st["c"]
    B, d = _kept(st, lambda B: B.BlockPlanDesc(c["requests"], st["blocks"], c["bs"], c["max_blocks"], st["table"].stride(0), st["free"].numel(), st["slots"].numel()))
    _must(B, B.ops_block_plan(d, st["cached"], st["added"], st["free"], st["table"], st["lengths"], st["starts"], st["slots"], st["counts"]))
    return st["table"], st["lengths"], st["starts"], st["slots"], st["counts"]


def _own_append(st):
    c = st["c"]
    row = st["kv_rows"].stride(0)
    B, d = _kept(st, lambda B: B.CacheAppendDesc(_layout(B, st), B.TYPES[c["type"]], c["tokens"], row, c["dim"], row, c["dim"]))
    _must(B, B.ops_cache_append(d, st["kv_rows"][:, 0], st["kv_rows"][:, 1], st["slots"], *st["pools"]))
    return tuple(st["pools"])


def _own_attend(st):
    c = st["c"]

    def make(B):
        d = B.PagedAttentionDesc(_layout(B, st), B.TYPES[c["type"]], c["requests"], c["kv"] * c["group"], st["table"].shape[1], st["table"].stride(0),
                                 st["longest"], c["window"], 1 / math.sqrt(c["dim"]), st["rows"].stride(0), c["dim"], st["out"].stride(0), c["dim"])
        st["workspace"] = torch.empty(B.ops_paged_attention_workspace(d), dtype=torch.uint8, device=DEV)
        return d
    B, d = _kept(st, make)
    _must(B, B.ops_paged_attention(d, st["rows"], *st["pools"], st["table"], st["lengths"], st["out"], st["lse"], st["workspace"]))
    return st["out"], st["lse"]


def _own_select(st):
    c = st["c"]

    def make(B):
        d = B.BeamSelectDesc(B.TYPES[c["type"]], c["requests"], c["beams"], c["vocab"], c["select"], 2, st["logits"].stride(0))
        st["workspace"] = torch.empty(B.ops_beam_select_workspace(d), dtype=torch.uint8, device=DEV)
        return d
    B, d = _kept(st, make)
    _must(B, B.ops_beam_select(d, st["logits"], st["scores"], st["ended"], st["best"], st["parents"], st["tokens"], st["workspace"]))
    return st["best"], st["parents"], st["tokens"]


def _own_reorder(st):
    c = st["c"]
    B, d = _kept(st, lambda B: B.BeamReorderDesc(_layout(B, st), c["rows"], c["rows"], st["table"].shape[1], st["table"].stride(0), st["table_out"].stride(0),
                                                 c["layers"], st["views"][0].stride(0)))
    _must(B, B.ops_beam_reorder(d, st["parents"], st["fill"], st["table"], st["spare"], st["table_out"], st["lengths_out"], *st["pools"]))
    return st["table_out"], st["lengths_out"], st["pools"][0], st["pools"][1]


# ---- the plain forms ---------------------------------------------------------------------------
def _plan(st):
    c = st["c"]
    bs, room, free = c["bs"], st["slots"].numel(), st["free"].numel()
    cached, added = st["cached"].long().clamp(min=0), st["added"].long().clamp(min=0)
    total = cached + added
    have, ends = (cached + bs - 1) // bs, added.cumsum(0)
    fits = (total <= c["max_blocks"] * bs) & (ends <= room)
    need = torch.where(fits, (total + bs - 1) // bs - have, 0)
    taken = need.cumsum(0)
    granted = fits & ((need == 0) | (taken <= free))
    need = torch.where(granted, need, 0)
    # the table: entry j of a granted request comes from the free list where it is new
    j = torch.arange(c["max_blocks"], device=DEV)[None, :] - have[:, None]
    new = (j >= 0) & (j < need[:, None])
    at = torch.where(new, (taken - need)[:, None] + j, 0)
    st["table"].copy_(torch.where(new, st["free"][at], st["table"]))
    st["lengths"].copy_(torch.where(granted, total, cached))
    st["starts"][1:] = ends.clamp(max=room).to(torch.int32)
    st["starts"][0] = 0
    # the slot map: the request of each new token, its place there, its block
    t = torch.arange(room, device=DEV)
    r = torch.searchsorted(ends, t, right=True)
    live = r < c["requests"]
    r = r.clamp(max=c["requests"] - 1)
    p = (cached + added - ends)[r] + t
    live = live & granted[r]
    p = torch.where(live, p, 0)
    block = st["table"][r, p // bs].long()
    live = live & (block >= 0) & (block < st["blocks"])
    st["slots"].copy_(torch.where(live, block * bs + p % bs, -1))
    st["counts"].copy_(torch.stack([torch.where(granted, taken, 0).amax(), ends[-1].clamp(max=room), (~granted).sum()]))
    return st["table"], st["lengths"], st["starts"], st["slots"], st["counts"]


def _append(st):
    slots = st["slots"].long()
    live = slots >= 0
    slots, bs = slots[live], st["c"]["bs"]
    k, v = st["views"]
    k[slots // bs, slots % bs] = st["kv_rows"][live, 0].to(k.dtype)
    v[slots // bs, slots % bs] = st["kv_rows"][live, 1].to(v.dtype)
    return tuple(st["pools"])


def _attend(st):
    c = st["c"]
    R, G, H, D = c["requests"], c["group"], c["kv"], c["dim"]
    t = torch.arange(st["longest"], device=DEV)
    lengths = st["lengths"].long()[:, None]
    block = st["table"].long()[:, t // c["bs"]]
    seen = (t < lengths) & (block >= 0) & (block < st["views"][0].shape[0])
    if c["window"]:
        seen = seen & (t >= lengths - c["window"])
    block = torch.where(seen, block, 0)
    k, v = (x[block, t % c["bs"]].permute(0, 2, 1, 3).float() for x in st["views"])   # [request][head][token][dim]
    q = st["rows"][:, :H * G].reshape(R, H, G, D).float()
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(D)
    seen = seen[:, None, None, :]
    s = s.masked_fill(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m.masked_fill(m == -math.inf, 0))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.masked_fill(~seen.transpose(-1, -2), 0)) / total
    st["out"].copy_(o.masked_fill(total == 0, 0).reshape(R, H * G, D))
    st["lse"].copy_((m + total.log()).reshape(R, H * G))
    return st["out"], st["lse"]


def _select(st):
    # in 64 bits: candidates of different beams lie next to each other
    c = st["c"]
    x = st["logits"].double()
    m = x.amax(-1, keepdim=True)
    s = st["scores"].double()[:, None] + (x - (m + torch.exp(x - m).sum(-1, keepdim=True).log()))
    if st["ended"] is not None:
        only = torch.where(torch.arange(c["vocab"], device=DEV)[None, :] == 2, st["scores"].double()[:, None], -math.inf)
        s = torch.where(st["ended"][:, None] != 0, only, s)
    s = torch.where(s < math.inf, s, -math.inf).reshape(c["requests"], -1)
    best, at = torch.sort(s, dim=-1, descending=True, stable=True)
    best, at = best[:, :c["select"]], at[:, :c["select"]]
    st["best"].copy_(best)
    st["parents"].copy_(at // c["vocab"] + torch.arange(c["requests"], device=DEV)[:, None] * c["beams"])
    st["tokens"].copy_(at % c["vocab"])
    return st["best"], st["parents"], st["tokens"]


def _reorder(st):
    c = st["c"]
    bs, p = c["bs"], st["parents"].long()
    n = st["fill"].long()[p]
    moved = (p != torch.arange(c["rows"], device=DEV)) & (n % bs != 0)
    table, j = st["table"][p], torch.arange(st["table"].shape[1], device=DEV)
    source, target = table.gather(1, (n // bs)[:, None])[:, 0].long(), st["spare"].long()
    table = torch.where(moved[:, None] & (j == (n // bs)[:, None]), st["spare"][:, None], table)
    st["table_out"].copy_(torch.where(j < ((n + bs - 1) // bs)[:, None], table, st["table_out"]))
    st["lengths_out"].copy_(n)
    row, token = (moved[:, None] & (torch.arange(bs, device=DEV) < (n % bs)[:, None])).nonzero(as_tuple=True)
    k, v = st["views"]
    k[:, target[row], token] = k[:, source[row], token]
    v[:, target[row], token] = v[:, source[row], token]
    return st["table_out"], st["lengths_out"], st["pools"][0], st["pools"][1]


# ---- the definitions in 64 bits ----------------------------------------------------------------
def exact(c, seed):
    st = prepare(c, seed)
    return {"plan": _exact_plan, "append": _exact_append, "attend": _exact_attend, "select": _exact_select, "reorder": _exact_reorder}[c["op"]](st)


def _exact_plan(st):
    return None     # whole numbers


def _exact_append(st):
    c = st["c"]
    pools = [p.double() for p in st["pools"]]
    slots = st["slots"].cpu().numpy()
    kept = np.flatnonzero(slots >= 0)
    where = torch.from_numpy(slots[kept].astype(np.int64)).to(DEV)
    rows = st["kv_rows"].double()[torch.from_numpy(kept).to(DEV)]
    for i, p in enumerate(pools):
        block, token = torch.div(where, c["bs"], rounding_mode="floor"), where.remainder(c["bs"])
        if c["order"] == "thd":
            p[block, token] = rows[:, i]
        else:
            p.transpose(1, 2)[block, token] = rows[:, i]
    return tuple(pools)


def _exact_attend(st):
    c = st["c"]
    out, lse = torch.zeros(st["out"].shape, dtype=torch.float64, device=DEV), torch.zeros(st["lse"].shape, dtype=torch.float64, device=DEV)
    table, lengths = st["table"].cpu().numpy(), st["lengths"].cpu().numpy()
    for r in range(c["requests"]):
        n = int(lengths[r])
        first = max(0, n - c["window"]) if c["window"] else 0
        places = np.arange(first, n)
        if not len(places):
            lse[r] = -math.inf
            continue
        block = torch.from_numpy(table[r, places // c["bs"]].astype(np.int64)).to(DEV)
        token = torch.from_numpy(places % c["bs"]).to(DEV)
        for h in range(c["kv"]):
            k, v = (x[block, token, h].double() for x in st["views"])
            mine = slice(h * c["group"], (h + 1) * c["group"])
            s = st["rows"][r, mine].double() @ k.t() * c["dim"] ** -0.5
            lse[r, mine] = torch.logsumexp(s, -1)
            out[r, mine] = torch.softmax(s, -1) @ v
    return out, lse


def _exact_select(st):
    c = st["c"]
    best, parents, tokens = [], [], []
    for r in range(c["requests"]):
        found = []
        for b in range(r * c["beams"], (r + 1) * c["beams"]):
            cum = float(st["scores"][b])
            if st["ended"] is not None and int(st["ended"][b]):
                if c["vocab"] > 2:
                    found.append((-cum, b, 2))
                continue
            x = st["logits"][b].double()
            top, at = torch.topk(x, min(c["vocab"], 8 * c["select"]))
            found += [(-s, b, t) for s, t in zip((cum + (top - torch.logsumexp(x, -1))).tolist(), at.tolist())]
        found = sorted(found)[:c["select"]]
        if len(found) < c["select"]:
            return None
        best.append([-f[0] for f in found])
        parents.append([f[1] for f in found])
        tokens.append([f[2] for f in found])
    return torch.tensor(best, dtype=torch.float64), torch.tensor(parents, dtype=torch.int32), torch.tensor(tokens, dtype=torch.int32)


def _exact_reorder(st):
    c = st["c"]
    table, fill, parents, spare = (st[k].cpu().numpy() for k in ("table", "fill", "parents", "spare"))
    pools = [p.double() for p in st["pools"]]
    new = np.full(table.shape, -1, np.int32)
    for i, p in enumerate(parents):
        full, rest = divmod(int(fill[p]), c["bs"])
        new[i, :full] = table[p, :full]
        if rest:
            new[i, full] = table[p, full] if p == i else spare[i]
            if p != i:
                for x in pools:
                    if c["order"] == "thd":
                        x[:, spare[i], :rest] = x[:, table[p, full], :rest]
                    else:
                        x[:, spare[i], :, :rest] = x[:, table[p, full], :, :rest]
    return torch.from_numpy(new), torch.from_numpy(fill[parents].astype(np.int32)), pools[0], pools[1]
