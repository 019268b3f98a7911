"""More operators of text generation that are timed: what a server of many requests asks for beside the steps of perf/operators.py.

A case is a dict of plain values; its "op" says which operator it calls.

  chunk    attention of the new tokens of all requests (prompts, pieces of prompts, single ones) over the paged cache
  scores   log probabilities of given tokens, their ranks, the entropy and the best alternatives
  sweep    uses of each block by the block tables, and the list of free blocks
  fork     requests that continue a part of another one, with full blocks shared
  compact  blocks in use moved to the front of the pool

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
        # five proposed tokens of one request looked over at once, the encoder's sizes (12 heads of 64, 32 bits) and its length: latency
        dict(name="chunk_1x5_f32", op="chunk", requests=1, kv=12, group=1, dim=64, bs=16, order="thd", type="f32", cache="f32",
             chunk=5, cached=379, spread=0, window=0, odd=0, mix=21),
        # a whole prompt, grouped heads
        dict(name="chunk_prompt_8191_bf16", op="chunk", requests=1, kv=8, group=4, dim=128, bs=16, order="thd", type="bf16", cache="bf16",
             chunk=8191, cached=0, spread=0, window=0, odd=0, mix=22),
        # pieces of long prompts over what is cached already, heads in front of tokens
        dict(name="chunk_3x509_over_40000_f16", op="chunk", requests=3, kv=8, group=8, dim=128, bs=64, order="htd", type="f16", cache="f16",
             chunk=509, cached=40000, spread=0, window=0, odd=0, mix=23),
        # a step in service: prompts, pieces and single tokens of many requests, one without tokens, one refused; 32 bits over a
        # 16-bit cache, odd block size, head size 80, a sliding window
        dict(name="chunk_24xmixed_f32_bf16", op="chunk", requests=24, kv=5, group=3, dim=80, bs=24, order="thd", type="f32", cache="bf16",
             chunk=600, cached=3000, spread=1, window=1000, odd=1, mix=24),
        # one sampled token at the encoder's vocabulary, an odd row length
        dict(name="scores_1_f32", op="scores", rows=1, vocab=30522, top=5, type="f32", pad=0),
        # all tokens of a prompt over a large odd vocabulary in half precision
        dict(name="scores_1000_bf16", op="scores", rows=1000, vocab=128257, top=20, type="bf16", pad=1),
        # a few requests' tables
        dict(name="sweep_8", op="sweep", rows=8, blocks=1024, bs=16, max_blocks=64, longest=1000, shared=0, mix=25),
        # thousands of requests, prefixes shared
        dict(name="sweep_4000", op="sweep", rows=4000, blocks=300001, bs=16, max_blocks=512, longest=8000, shared=1, mix=26),
        # three more samples of one request
        dict(name="fork_3", op="fork", forks=3, rows=8, layers=12, kv=12, dim=64, bs=16, order="thd", cache="f32", longest=384, short=0, mix=27),
        # eight samples of each of 32 requests through all layers of a larger model; blocks run out
        dict(name="fork_224", op="fork", forks=224, rows=256, layers=24, kv=8, dim=128, bs=16, order="htd", cache="bf16", longest=1500, short=1, mix=28),
        # a small pool
        dict(name="compact_64", op="compact", rows=6, blocks=64, layers=12, kv=12, dim=64, bs=16, order="thd", cache="f32", longest=200, shared=0, mix=29),
        # a pool of a larger model, half of it in use
        dict(name="compact_1500", op="compact", rows=64, blocks=1500, layers=24, kv=8, dim=128, bs=16, order="thd", cache="bf16", longest=700, shared=1, mix=30),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("chunk", "chunk", "chunk", "chunk", "scores", "scores", "sweep", "fork", "compact"))
    mix = rng.randrange(1, 1 << 20)
    bs = rng.choice((8, 16, 16, 24, 32, 64, 128))
    dim = rng.choice((32, 40, 64, 64, 72, 80, 96, 128, 128, 128, 192, 256))
    kv = rng.choice((1, 2, 4, 5, 8, 12))
    order = rng.choice(("thd", "htd"))
    pair = rng.choice((("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "bf16")))
    if op == "sweep":
        return dict(op=op, rows=_log_int(rng, 1, 4000), blocks=_log_int(rng, 64, 300000), bs=bs, max_blocks=_log_int(rng, 16, 512), longest=_log_int(rng, 8, 8000),
                    shared=rng.choice((0, 1)), mix=mix)
    while op == "scores":
        c = dict(op=op, rows=_log_int(rng, 1, 2000), vocab=_log_int(rng, 300, 152000), top=rng.choice((0, 1, 2, 5, 8, 20, 32)), type=pair[0], pad=rng.choice((0, 1)))
        if c["rows"] * c["vocab"] < 1.2e8:
            return c
    while op == "fork":
        c = dict(op=op, forks=_log_int(rng, 1, 200), rows=0, layers=rng.choice((1, 6, 12, 24)), kv=kv, dim=dim, bs=rng.choice((8, 16, 24, 32)), order=order,
                 cache=pair[1], longest=_log_int(rng, 8, 1500), short=rng.choice((0, 1)), mix=mix)
        c["rows"] = c["forks"] + _log_int(rng, 1, 64)
        if (c["rows"] + c["forks"] + 64) * c["layers"] * kv * dim * c["bs"] < 3e8:
            return c
    while op == "compact":
        c = dict(op=op, rows=_log_int(rng, 1, 64), blocks=_log_int(rng, 16, 3000), layers=rng.choice((1, 6, 12, 24)), kv=kv, dim=dim, bs=rng.choice((8, 16, 24, 32)),
                 order=order, cache=pair[1], longest=0, shared=rng.choice((0, 1)), mix=mix)
        c["longest"] = _log_int(rng, 8, min(1500, c["blocks"] * c["bs"] // 2))
        if c["blocks"] * c["layers"] * kv * dim * c["bs"] < 4e8:
            return c
    while True:
        c = dict(op=op, requests=_log_int(rng, 1, 32), kv=kv, group=rng.choice((1, 1, 2, 3, 4, 7, 8, 16, 20)), dim=dim, bs=bs, order=order, type=pair[0],
                 cache=pair[1], chunk=_log_int(rng, 1, 4000), cached=_log_int(rng, 1, 40000) - 1, spread=rng.choice((0, 1, 1)),
                 window=rng.choice((0, 0, 0, _log_int(rng, 1, 4000))), odd=rng.choice((0, 1)), mix=mix)
        both = c["chunk"] + c["cached"]
        if c["requests"] * kv * c["group"] * c["chunk"] * both < 1e9 and c["requests"] * kv * both * dim < 2.5e8:
            return c


# ---- what a case says about lengths ------------------------------------------------------------
def _chunks(c):
    """(cached, added, granted) of each request: the case's lengths, or spread below them over the logarithm; "odd": one without new tokens
    and one that the block plan refused, where there are others."""
    r = random.Random(c["mix"])
    n = c["requests"]
    cached = [_log_int(r, 1, c["cached"] + 1) - 1 if c["spread"] else c["cached"] for _ in range(n)]
    added = [_log_int(r, 1, c["chunk"]) if c["spread"] else c["chunk"] for _ in range(n)]
    most = r.randrange(n)
    cached[most], added[most] = c["cached"], c["chunk"]
    granted = [True] * n
    if c["odd"] and n > 2:
        added[(most + 1) % n] = 0
        granted[(most + 2) % n] = False
    return cached, added, granted


def _rows_of_tables(c):
    """Lengths of the rows of a block table, and how many leading blocks each shares with the row before it."""
    r = random.Random(c["mix"])
    n = [_log_int(r, 1, c["longest"]) for _ in range(c["rows"])]
    bs, shared = c["bs"], [0] * c["rows"]
    for i in range(1, c["rows"]):
        if r.random() < 0.1:
            n[i] = 0
        if c["shared"] and i % 4:
            shared[i] = min(n[i], n[i - 1]) // bs
    return n, shared


def _tables(c):
    """(lengths, the blocks that each row has of its own and shares, blocks in use): rows that do not fit into the pool any more have length 0."""
    n, shared = _rows_of_tables(c)
    most, used = c["blocks"] * 9 // 10, 0
    room = c.get("max_blocks", -(-c["longest"] // c["bs"]))
    for i in range(len(n)):
        n[i] = min(n[i], room * c["bs"])
        have = -(-n[i] // c["bs"])
        shared[i] = min(shared[i], have, -(-n[i - 1] // c["bs"]) if i else 0)
        if used + have - shared[i] > most:
            n[i], shared[i], have = 0, 0, 0
        used += have - shared[i]
    return n, shared, used


def _forks(c):
    """(lengths of the parents' rows, parent of each fork, tokens of each fork): the first rows are parents, the last ones children."""
    r = random.Random(c["mix"])
    base = c["rows"] - c["forks"]
    n = [_log_int(r, 1, c["longest"]) for _ in range(base)]
    parents = [i % base for i in range(c["forks"])]
    return n, parents, [n[p] if r.random() < 0.7 else r.randrange(n[p] + 1) for p in parents]


def _fork_needs(c):
    n, parents, tokens = _forks(c)
    need = [t % c["bs"] != 0 for t in tokens]
    return need, (max(1, sum(need) * 7 // 8) if c["short"] else sum(need) + 4)


def _seen(p, window):
    """Sum over a run of places [p0, p1) of the tokens that each sees."""
    p0, p1 = p
    upto = lambda m: m * (m + 1) // 2                                                                          # noqa: E731
    if not window:
        return upto(p1) - upto(p0)
    a, b = min(p0, window), min(p1, window)
    return upto(b) - upto(a) + window * (p1 - p0 - (b - a))


def work(c):
    op = c["op"]
    if op == "chunk":
        cached, added, granted = _chunks(c)
        heads, e = c["kv"] * c["group"], BYTES[c["type"]]
        read = sum(a + b - (max(0, a + 1 - c["window"]) if c["window"] else 0) for a, b, g in zip(cached, added, granted) if g and b)
        seen = sum(_seen((a, a + b), c["window"]) for a, b, g in zip(cached, added, granted) if g)
        return {"bytes": 2 * read * c["kv"] * c["dim"] * BYTES[c["cache"]] + sum(added) * heads * (2 * c["dim"] * e + 4) + 4 * -(-read // c["bs"]) + 12 * c["requests"],
                "flops": 4 * seen * heads * c["dim"]}
    if op == "scores":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * BYTES[c["type"]] + c["rows"] * (16 + 8 * c["top"]), "flops": 6 * n}
    if op == "sweep":
        n, _, used = _tables(c)
        return {"bytes": 4 * (c["rows"] + sum(-(-m // c["bs"]) for m in n) + c["blocks"] + c["blocks"] - used + 3), "flops": 0}
    block = c["layers"] * c["kv"] * c["dim"] * BYTES[c["cache"]]       # of one token, keys alone
    if op == "fork":
        _, _, tokens = _forks(c)
        need, room = _fork_needs(c)
        moved, entries, taken = 0, 0, 0
        for t, x in zip(tokens, need):
            taken += x
            if not x or taken <= room:
                moved, entries = moved + (t % c["bs"] if x else 0), entries + -(-t // c["bs"])
        return {"bytes": 4 * moved * block + 8 * entries + 16 * c["forks"], "flops": 0}
    n, _, used = _tables(c)
    moved = _moved(c)
    return {"bytes": 4 * moved * c["bs"] * block + 8 * sum(-(-m // c["bs"]) for m in n) + 4 * c["rows"], "flops": 0}


def _moved(c):
    """Blocks that a compaction moves: those in use behind the first `used` (which blocks are in use is the case's, which row has them the seed's)."""
    used = _tables(c)[2]
    return int((_in_use(c, used) >= used).sum())


def _in_use(c, used):
    return np.random.default_rng(c["mix"]).permutation(c["blocks"])[:used].astype(np.int32)


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


def _fill_tables(c, cpu, width):
    """Tables of _tables()'s rows.  Which blocks are in use is the case's for a compaction, whose work it is, and the seed's for a sweep."""
    n, shared, used = _tables(c)
    mine = cpu.permutation(_in_use(c, used) if c["op"] == "compact" else c["blocks"])[:used].astype(np.int32)
    table, at = np.full((c["rows"], width), -1, np.int32), 0
    for i, m in enumerate(n):
        have = -(-m // c["bs"])
        if shared[i]:
            table[i, :shared[i]] = table[i - 1, :shared[i]]
        table[i, shared[i]:have] = mine[at:at + have - shared[i]]
        at += have - shared[i]
    return n, table


def prepare(c, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    cpu = np.random.default_rng(seed)
    st = {"c": c}
    op = c["op"]
    if op == "chunk":
        cached, added, granted = _chunks(c)
        lengths = [a + b if g else a for a, b, g in zip(cached, added, granted)]
        have = [-(-n // c["bs"]) for n in lengths]
        width = max(1, max(have))
        order = cpu.permutation(sum(have) + 3).astype(np.int32)
        table = np.full((c["requests"], width), -1, np.int32)
        table[np.arange(width)[None, :] < np.asarray(have)[:, None]] = order[:sum(have)]
        st["pools"], st["views"] = _pools(c, len(order), gen)
        heads, tokens = c["kv"] * c["group"], sum(added) + (7 if c["odd"] else 0)      # (a batch padded to a size)
        # the queries' part of a row that holds keys and values behind them
        st["rows"] = _normal((tokens, heads + 2 * c["kv"], c["dim"]), c["type"], gen) * 1.5
        st.update(table=torch.from_numpy(table).to(DEV), starts=_ints(np.concatenate([[0], np.cumsum(added)]).tolist()), cached=_ints(cached), lengths=_ints(lengths),
                  longest=max(1, max(lengths)), out=torch.zeros((tokens, heads, c["dim"]), dtype=DTYPES[c["type"]], device=DEV),
                  lse=torch.zeros((tokens, heads), dtype=torch.float32, device=DEV))
    elif op == "scores":
        st["logits"] = (_normal((c["rows"], c["vocab"]), "f32", gen) * 2.5).to(DTYPES[c["type"]])
        tokens = torch.randint(0, c["vocab"], (c["rows"],), generator=gen, device=DEV, dtype=torch.int32)
        # half of them as a model would have them
        tokens = torch.where(torch.rand((c["rows"],), generator=gen, device=DEV) < 0.5, st["logits"].argmax(-1).to(torch.int32), tokens)
        if c["pad"]:
            tokens[-1] = -1
        st.update(tokens=tokens, scores=torch.zeros(c["rows"], device=DEV), ranks=torch.zeros(c["rows"], dtype=torch.int32, device=DEV),
                  entropy=torch.zeros(c["rows"], device=DEV), top_tokens=torch.zeros((c["rows"], c["top"]), dtype=torch.int32, device=DEV),
                  top_scores=torch.zeros((c["rows"], c["top"]), device=DEV))
    elif op == "sweep":
        n, table = _fill_tables(c, cpu, c["max_blocks"])
        st.update(lengths=_ints(n), table=torch.from_numpy(table).to(DEV), uses=_ints([0] * c["blocks"]), free=_ints([-1] * c["blocks"]), counts=_ints([0, 0, 0]))
    elif op == "fork":
        n, parents, tokens = _forks(c)
        _, room = _fork_needs(c)
        width = -(-c["longest"] // c["bs"]) + 1
        used = max(64, 2 * c["rows"])
        order = cpu.permutation(used + room).astype(np.int32)
        st["pools"], st["views"] = _pools(c, len(order), gen, c["layers"])
        st.update(parents=_ints(parents), children=_ints(list(range(c["rows"] - c["forks"], c["rows"]))), tokens=_ints(tokens), lengths=_ints(n + [0] * c["forks"]),
                  free=torch.from_numpy(order[used:].copy()).to(DEV), table=torch.from_numpy(order[cpu.integers(0, used, (c["rows"], width))]).to(DEV),
                  counts=_ints([0, 0]))
    else:
        width = -(-c["longest"] // c["bs"])
        n, table = _fill_tables(c, cpu, width)
        st["pools"], st["views"] = _pools(c, c["blocks"], gen, c["layers"])
        st.update(lengths=_ints(n), table=torch.from_numpy(table).to(DEV), table_out=torch.full((c["rows"], width), -1, dtype=torch.int32, device=DEV), counts=_ints([0, 0]))
    if op in ("chunk", "fork", "compact"):
        v = st["views"][0]
        st["strides"] = (v.stride(-4), v.stride(-3), v.stride(-2))
    return st


def run(st):
    op = st["c"]["op"]
    if own:
        return {"chunk": _own_chunk, "scores": _own_scores, "sweep": _own_sweep, "fork": _own_fork, "compact": _own_compact}[op](st)
    return {"chunk": _chunk, "scores": _scores, "sweep": _sweep, "fork": _fork, "compact": _compact}[op](st)


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


def _workspace(nbytes):
    return torch.empty(nbytes, dtype=torch.uint8, device=DEV) if nbytes else None


def _own_chunk(st):
    c = st["c"]

    def make(B):
        d = B.ChunkAttentionDesc(_layout(B, st), B.TYPES[c["type"]], c["requests"], c["kv"] * c["group"], st["rows"].shape[0], st["table"].shape[1],
                                 st["table"].stride(0), st["longest"], c["window"], 1 / math.sqrt(c["dim"]), st["rows"].stride(0), c["dim"], st["out"].stride(0), c["dim"])
        st["workspace"] = _workspace(B.ops_chunk_attention_workspace(d))
        return d
    B, d = _kept(st, make)
    _must(B, B.ops_chunk_attention(d, st["rows"], *st["pools"], st["table"], st["starts"], st["cached"], st["lengths"], st["out"], st["lse"], st["workspace"]))
    return st["out"], st["lse"]


def _own_scores(st):
    c = st["c"]

    def make(B):
        d = B.TokenScoresDesc(B.TYPES[c["type"]], c["rows"], c["vocab"], c["top"], st["logits"].stride(0))
        st["workspace"] = _workspace(B.ops_token_scores_workspace(d))
        return d
    B, d = _kept(st, make)
    top = (st["top_tokens"], st["top_scores"]) if c["top"] else (None, None)
    _must(B, B.ops_token_scores(d, st["logits"], st["tokens"], st["scores"], st["ranks"], st["entropy"], *top, st["workspace"]))
    return st["scores"], st["ranks"], st["entropy"], st["top_tokens"], st["top_scores"]


def _own_sweep(st):
    c = st["c"]

    def make(B):
        d = B.BlockSweepDesc(c["rows"], c["blocks"], c["bs"], c["max_blocks"], st["table"].stride(0))
        st["workspace"] = _workspace(B.ops_block_sweep_workspace(d))
        return d
    B, d = _kept(st, make)
    _must(B, B.ops_block_sweep(d, st["table"], st["lengths"], st["uses"], st["free"], st["counts"], st["workspace"]))
    return st["uses"], st["free"], st["counts"]


def _own_fork(st):
    c = st["c"]
    B, d = _kept(st, lambda B: B.CacheForkDesc(_layout(B, st), c["forks"], c["rows"], st["table"].shape[1], st["table"].stride(0), st["free"].numel(), c["layers"],
                                               st["views"][0].stride(0)))
    _must(B, B.ops_cache_fork(d, st["parents"], st["children"], st["tokens"], st["free"], st["table"], st["lengths"], st["counts"], *st["pools"]))
    return st["table"], st["lengths"], st["counts"], st["pools"][0], st["pools"][1]


def _own_compact(st):
    c = st["c"]

    def make(B):
        d = B.CacheCompactDesc(_layout(B, st), c["rows"], st["table"].shape[1], st["table"].stride(0), st["table_out"].stride(0), c["layers"], st["views"][0].stride(0))
        st["workspace"] = _workspace(B.ops_cache_compact_workspace(d))
        return d
    B, d = _kept(st, make)
    _must(B, B.ops_cache_compact(d, st["table"], st["lengths"], st["table_out"], st["counts"], *st["pools"], st["workspace"]))
    return st["table_out"], st["counts"], st["pools"][0], st["pools"][1]


# ---- the plain forms ---------------------------------------------------------------------------
def _chunk(st):
    c = st["c"]
    R, G, H, D, C = c["requests"], c["group"], c["kv"], c["dim"], c["chunk"]
    t = torch.arange(st["longest"], device=DEV)
    lengths, starts = st["lengths"].long(), st["starts"].long()
    block = st["table"].long()[:, t // c["bs"]]
    there = (t < lengths[:, None]) & (block >= 0) & (block < st["views"][0].shape[0])
    block = torch.where(there, block, 0)
    k, v = (x[block, t % c["bs"]].permute(0, 2, 1, 3).float() for x in st["views"])   # [request][head][token][dim]
    i = torch.arange(C, device=DEV)
    mine = i < (starts[1:] - starts[:-1])[:, None]                                    # [request][new token]
    token = torch.where(mine, starts[:-1, None] + i, 0)
    place = (st["cached"].long()[:, None] + i)[:, :, None]
    seen = there[:, None, :] & (t <= place) & (place < lengths[:, None, None])
    if c["window"]:
        seen = seen & (t > place - c["window"])
    q = st["rows"][token, :H * G].reshape(R, C, H, G, D).permute(0, 2, 3, 1, 4).reshape(R, H, G * C, D).float()
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(D)).reshape(R, H, G, C, -1)
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(m.masked_fill(m == -math.inf, 0)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(R, H, G * C, -1), v.masked_fill(~there[:, None, :, None], 0)).reshape(R, H, G, C, D) / total
    o = o.masked_fill(total == 0, 0)
    st["out"][token[mine]] = o.permute(0, 3, 1, 2, 4).reshape(R, C, H * G, D)[mine].to(st["out"].dtype)
    st["lse"][token[mine]] = (m + total.log()).permute(0, 3, 1, 2, 4).reshape(R, C, H * G)[mine]
    return st["out"], st["lse"]


def _scores(st):
    c = st["c"]
    x = st["logits"].float()
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    near = x - m                               # (scores are differences from the maximum, less the logarithm)
    log = total.log()
    token = st["tokens"].long()[:, None]
    given = (token >= 0) & (token < c["vocab"])
    at = torch.where(given, token, 0)
    value = x.gather(1, at)
    before = ((x > value) | ((x == value) & (torch.arange(c["vocab"], device=DEV) < at))).sum(-1, keepdim=True)
    st["scores"].copy_(torch.where(given, near.gather(1, at) - log, -math.inf)[:, 0])
    st["ranks"].copy_(torch.where(given, before, -1)[:, 0])
    st["entropy"].copy_((log - (e * near).sum(-1, keepdim=True) / total)[:, 0])
    best, at = torch.sort(x, dim=-1, descending=True, stable=True)
    st["top_tokens"].copy_(at[:, :c["top"]])
    st["top_scores"].copy_(best[:, :c["top"]] - m - log)
    return st["scores"], st["ranks"], st["entropy"], st["top_tokens"], st["top_scores"]


def _used_entries(st):
    """Which entries of the table count, and their blocks; [row][entry]."""
    bs = st["c"]["bs"]
    n = ((st["lengths"].long() + bs - 1) // bs)[:, None]
    return torch.arange(st["table"].shape[1], device=DEV) < n, st["table"].long()


def _sweep(st):
    c = st["c"]
    counted, block = _used_entries(st)
    inside = counted & (block >= 0) & (block < c["blocks"])
    block = block[inside]
    st["uses"].zero_().index_add_(0, block, torch.ones_like(block, dtype=torch.int32))
    free = st["uses"] == 0
    rank = free.cumsum(0)
    listed_at = torch.cat([st["free"], st["free"][:1]])                              # (one more entry for those that are in use)
    listed_at[torch.where(free, rank - 1, c["blocks"])] = torch.arange(c["blocks"], dtype=torch.int32, device=DEV)
    st["free"].copy_(listed_at[:-1])
    st["counts"].copy_(torch.stack([rank[-1], c["blocks"] - rank[-1], (counted & ~inside).sum()]))
    return st["uses"], st["free"], st["counts"]


def _fork(st):
    c = st["c"]
    bs, p, child = c["bs"], st["parents"].long(), st["children"].long()
    n = torch.minimum(st["tokens"], st["lengths"][p]).long()
    need = n % bs != 0
    taken = need.cumsum(0)
    granted = ~need | (taken <= st["free"].numel())
    target = st["free"].long()[torch.where(need & granted, taken - 1, 0)]
    rows, j = st["table"][p], torch.arange(st["table"].shape[1], device=DEV)
    source = rows.gather(1, (n // bs)[:, None])[:, 0].long()
    rows = torch.where(need[:, None] & (j == (n // bs)[:, None]), target[:, None].int(), rows)
    st["table"][child] = torch.where(granted[:, None] & (j < ((n + bs - 1) // bs)[:, None]), rows, st["table"][child])
    st["lengths"][child] = torch.where(granted, n, st["lengths"][child].long()).int()
    st["counts"].copy_(torch.stack([taken[-1].clamp(max=st["free"].numel()), (~granted).sum()]))
    row, token = ((need & granted)[:, None] & (torch.arange(bs, device=DEV) < (n % bs)[:, None])).nonzero(as_tuple=True)
    k, v = st["views"]
    k[:, target[row], token] = k[:, source[row], token]
    v[:, target[row], token] = v[:, source[row], token]
    return st["table"], st["lengths"], st["counts"], st["pools"][0], st["pools"][1]


def _compact(st):
    c = st["c"]
    counted, block = _used_entries(st)
    used = torch.zeros(c["blocks"], dtype=torch.bool, device=DEV)
    used[block[counted]] = True
    n, number = used.sum(), torch.arange(c["blocks"], device=DEV)
    # the last block in use goes to the first free one, the last but one to the second
    source, target = (used & (number >= n)).nonzero()[:, 0].flip(0), (~used & (number < n)).nonzero()[:, 0]
    to = number.clone()
    to[source] = target
    st["table_out"].copy_(torch.where(counted, to[torch.where(counted, block, 0)], st["table_out"].long()))
    st["counts"].copy_(torch.stack([n, (used & (number >= n)).sum()]))
    for x in st["pools"]:
        x[:, target] = x[:, source]
    return st["table_out"], st["counts"], st["pools"][0], st["pools"][1]


# ---- the definitions in 64 bits ----------------------------------------------------------------
def exact(c, seed):
    st = prepare(c, seed)
    return {"chunk": _exact_chunk, "scores": _exact_scores, "sweep": _exact_sweep, "fork": _exact_fork, "compact": _exact_compact}[c["op"]](st)


def _exact_chunk(st):
    c = st["c"]
    out, lse = torch.zeros(st["out"].shape, dtype=torch.float64, device=DEV), torch.zeros(st["lse"].shape, dtype=torch.float64, device=DEV)
    table, starts, cached, lengths = (st[k].cpu().numpy() for k in ("table", "starts", "cached", "lengths"))
    for r in range(c["requests"]):
        first, added, n = int(starts[r]), int(starts[r + 1] - starts[r]), int(lengths[r])
        if not added:
            continue
        if n < cached[r] + added:
            lse[first:first + added] = -math.inf
            continue
        places = np.arange(n)
        block = torch.from_numpy(table[r, places // c["bs"]].astype(np.int64)).to(DEV)
        token = torch.from_numpy(places % c["bs"]).to(DEV)
        far = torch.arange(n, device=DEV)[None, :] - torch.arange(int(cached[r]), n, device=DEV)[:, None]        # key's place less the query's
        hidden = far > 0
        if c["window"]:
            hidden = hidden | (far <= -c["window"])
        for h in range(c["kv"]):
            k, v = (x[block, token, h].double() for x in st["views"])
            for g in range(h * c["group"], (h + 1) * c["group"]):
                s = st["rows"][first:first + added, g].double() @ k.t() * c["dim"] ** -0.5
                s[hidden] = -math.inf
                lse[first:first + added, g] = torch.logsumexp(s, -1)
                out[first:first + added, g] = torch.softmax(s, -1) @ v
    return out, lse


def _exact_scores(st):
    c = st["c"]
    scores, entropy = torch.zeros(c["rows"], dtype=torch.float64, device=DEV), torch.zeros(c["rows"], dtype=torch.float64, device=DEV)
    best = torch.zeros((c["rows"], c["top"]), dtype=torch.float64, device=DEV)
    for r in range(c["rows"]):
        logp = torch.log_softmax(st["logits"][r].double(), -1)
        token = int(st["tokens"][r])
        scores[r] = logp[token] if 0 <= token < c["vocab"] else -math.inf
        entropy[r] = -(logp.exp() * logp).sum()
        best[r] = torch.topk(logp, c["top"]).values
    return scores, None, entropy, None, best


def _exact_sweep(st):
    return None     # whole numbers


def _move(c, pool, source, target, tokens):
    """The first `tokens` of a block to another, in all layers."""
    if c["order"] == "thd":
        pool[:, target, :tokens] = pool[:, source, :tokens]
    else:
        pool[:, target, :, :tokens] = pool[:, source, :, :tokens]


def _exact_fork(st):
    c = st["c"]
    table, lengths, parents, children, tokens, free = (st[k].cpu().numpy().copy() for k in ("table", "lengths", "parents", "children", "tokens", "free"))
    pools = [p.double() for p in st["pools"]]
    used = refused = 0
    for p, i, n in zip(parents, children, tokens):
        full, rest = divmod(int(min(n, lengths[p])), c["bs"])
        if rest and used == len(free):
            refused += 1
            continue
        table[i, :full], lengths[i] = table[p, :full], full * c["bs"] + rest
        if rest:
            table[i, full] = free[used]
            for x in pools:
                _move(c, x, int(table[p, full]), int(free[used]), rest)
            used += 1
    return torch.from_numpy(table), torch.from_numpy(lengths), torch.tensor([used, refused], dtype=torch.int32), pools[0], pools[1]


def _exact_compact(st):
    c = st["c"]
    table, lengths = st["table"].cpu().numpy(), st["lengths"].cpu().numpy()
    pools = [p.double() for p in st["pools"]]
    used = sorted({int(b) for row, n in zip(table, lengths) for b in row[:-(-n // c["bs"])]})
    holes = sorted(set(range(len(used))) - set(used))
    to = dict(zip(used[::-1], holes))
    for b, t in to.items():
        for x in pools:
            _move(c, x, b, t, c["bs"])
    new = np.full(table.shape, -1, np.int32)
    for i, n in enumerate(lengths):
        for j in range(-(-n // c["bs"])):
            new[i, j] = to.get(int(table[i, j]), int(table[i, j]))
    return torch.from_numpy(new), torch.tensor([len(used), len(holes)], dtype=torch.int32), pools[0], pools[1]
