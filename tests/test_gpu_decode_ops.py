"""The operators of text generation on the device against plain forms in 64 bits (tests/decode_ref.py): block tables and slot maps,
cache writes, attention over a paged cache, beam search, and a run of them together."""
import ctypes

import numpy as np
import pytest

from reef_amd import binding as B
from tests import decode_ref as R
from tests.decode_ref import BF16, F16, F32, HALF

pytestmark = pytest.mark.gpu


def up(a):
    return B.DeviceBuffer.from_array(np.ascontiguousarray(a)) if np.asarray(a).size else B.DeviceBuffer(16)


def ok(status):
    assert status == 0, B.last_error()


def ints(a):
    return up(np.asarray(a, np.int32))


class Pools:
    """Key and value pools on the host (float64 values as the device has them) and on the device, in either order of heads and tokens,
    with `pad` unused elements behind each innermost row group."""

    def __init__(self, kind, blocks, bs, kv, dim, order="thd", pad=0, layers=None, seed=0, size=1.0):
        rng = np.random.default_rng(seed)
        if order == "thd":
            head, slot = dim, kv * dim + pad
            block = bs * slot
        else:
            slot, head = dim, bs * dim + pad
            block = kv * head
        self.kind, self.shape, self.per_layer = kind, (blocks, bs, kv, dim), blocks * block
        self.layers = layers
        n = self.per_layer * (layers or 1)
        self.raw = [R.encode((rng.standard_normal(n) * size).astype(np.float32), kind) for _ in range(2)]
        self.layout = B.CacheLayout(kind, blocks, bs, kv, dim, block, slot, head)
        self.strides = (block, slot, head, 1)
        self.send()

    def send(self):
        self.dev = [up(r) for r in self.raw]

    def view(self, raw, layer=0):
        """[block][token][head][dim] of a raw pool, writable."""
        size = raw.itemsize
        return np.lib.stride_tricks.as_strided(raw[layer * self.per_layer:], self.shape, [s * size for s in self.strides])

    def values(self, i):
        return R.decode(self.view(self.raw[i]), self.kind)

    def fetch(self):
        return [d.to_array(R.np_type(self.kind)) for d in self.dev]


# ---- block tables and slot maps -----------------------------------------------------------------
def run_plan(cached, added, free, table, blocks, bs, max_blocks, max_tokens):
    n, stride = len(cached), table.shape[1]
    d = B.BlockPlanDesc(n, blocks, bs, max_blocks, stride, len(free), max_tokens)
    # a word behind each output, to be left alone
    out = [ints(np.full(k + 1, -7)) for k in (n, n + 1, max_tokens, 3)]
    t = up(np.concatenate([table.ravel(), [-7]]).astype(np.int32))
    for _ in range(2):                       # a second call over its own results: nothing is added up
        ok(B.ops_block_plan(d, ints(cached), ints(added), ints(free), t, *out))
    got = [t] + out
    got = [g.to_array(np.int32) for g in got]
    assert all(g[-1] == -7 for g in got)
    want = R.plan(cached, added, free, table, blocks, bs, max_blocks, max_tokens)
    for g, w, what in zip(got, want, ("table", "lengths", "starts", "slots", "counts")):
        np.testing.assert_array_equal(g[:-1], np.asarray(w).ravel(), what)


def plan_case(rng, n, bs, max_blocks, longest, added, stride=None):
    cached = rng.integers(0, longest, n)
    cached = np.minimum(cached, max_blocks * bs)
    more = rng.integers(0, added + 1, n)
    stride = stride or max_blocks
    table = np.full((n, stride), -1, np.int64)
    for i, c in enumerate(cached):
        have = min(-(-int(c) // bs), max_blocks)
        table[i, :have] = rng.integers(0, 5000, have)
    return cached, more, table


@pytest.mark.parametrize("n", [0, 1, 2, 63, 255, 257, 1023, 1024, 1025, 3000])
@pytest.mark.parametrize("bs,added", [(16, 1), (1, 3), (24, 100), (128, 1)])
def test_plan(n, bs, added):
    rng = np.random.default_rng(n * 131 + bs)
    cached, more, table = plan_case(rng, n, bs, 40, 300, added, stride=43)
    need = int(sum(-(-(c + a) // bs) - -(-c // bs) for c, a in zip(cached, more)))
    for free, room in ((need + 3, int(more.sum()) + 5), (need * 2 // 3, int(more.sum())), (need, int(more.sum()) * 3 // 4), (0, int(more.sum()) + 1), (need, 0)):
        run_plan(cached, more, rng.permutation(5000)[:free], table, 5000, bs, 40, room)


def test_plan_odd_requests():
    rng = np.random.default_rng(5)
    # negative lengths, rows that are full, nothing to add, a huge wish, a block that is not one of the pool's
    cached = np.array([-3, 64, 63, 10, 0, 5, 17, -2 ** 31, 2 ** 31 - 1, 64])
    more = np.array([2, 1, 1, 0, 64, 2 ** 31 - 1, 3, 5, 1, 0])
    table = np.full((10, 4), -1, np.int64)
    table[6, :2] = [4, 77]
    table[2, :4] = [1, 2, 3, -5]
    table[3, 0] = 8
    for room in (2 ** 20, 80):
        run_plan(cached, more, rng.permutation(20), table, 20, 16, 4, room)
    run_plan(np.zeros(600, int), np.full(600, 2 ** 31 - 1), np.arange(20), np.full((600, 4), -1), 20, 16, 4, 100)
    run_plan(np.array([15]), np.array([0]), np.arange(0), np.full((1, 1), 3), 20, 16, 1, 0)
    # one request with a very long prompt among decode steps
    cached, more = np.full(300, 31), np.ones(300, int)
    more[150] = 100000
    run_plan(cached, more, rng.permutation(9000), np.full((300, 7000), 2), 9000, 16, 7000, 110000)


# ---- cache writes -------------------------------------------------------------------------------
@pytest.mark.parametrize("kind,cache", [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("order,bs,kv,dim,tokens,pad", [("thd", 16, 8, 128, 1, 0), ("htd", 32, 12, 64, 77, 8), ("thd", 1, 1, 8, 9, 0),
                                                        ("htd", 24, 5, 80, 700, 0), ("thd", 7, 3, 256, 33, 16)])
def test_append(kind, cache, order, bs, kv, dim, tokens, pad):
    rng = np.random.default_rng(tokens)
    blocks = -(-tokens // bs) + 5
    pools = Pools(cache, blocks, bs, kv, dim, order, pad)
    extra = 8
    rows = (rng.standard_normal((tokens, 2, kv, dim + extra)) * 3).astype(np.float32)
    # as they round: infinities, NaN, over the 16-bit float's range and on its border, subnormal in it, halfway, subnormal in 32 bits
    rows[0, :, 0, :8] = [np.inf, -np.inf, np.nan, 1e30, 65519.9, 3e-6, 2.0 ** -25 * 3, 1e-39]
    rows = R.encode(rows, kind)
    slots = rng.permutation(blocks * bs)[:tokens].astype(np.int64)
    slots[rng.random(tokens) < 0.1] = -1
    if tokens > 4:
        slots[3], slots[4] = blocks * bs, 2 ** 31 - 1         # behind the pool
    slots[0] = 1 if 1 < blocks * bs and 1 not in slots[1:] else slots[0]
    row = 2 * kv * (dim + extra)
    d = B.CacheAppendDesc(pools.layout, kind, tokens, row, dim + extra, row, dim + extra)
    dev = up(rows)
    size = rows.itemsize
    ok(B.ops_cache_append(d, dev.ptr.value, dev.ptr.value + kv * (dim + extra) * size, ints(slots), *pools.dev))
    want = [r.copy() for r in pools.raw]
    for i in range(2):
        v = pools.view(want[i])
        for t, s in enumerate(slots):
            if 0 <= s < blocks * bs:
                x = rows[t, i, :, :dim]
                v[s // bs, s % bs] = x if kind == cache else R.encode(x.astype(np.float32), cache)
    for got, w in zip(pools.fetch(), want):
        g, w = R.decode(got, cache), R.decode(w, cache)
        np.testing.assert_array_equal(g, w)                    # (one NaN is as good as another)


# ---- attention ----------------------------------------------------------------------------------
def run_attend(kind, cache, order, bs, kv, group, dim, lengths, window=0, pad=0, scale=None, longest=0, seed=0, spoil=True, bad=0.0, q_pad=0, grow=1.0,
               max_blocks=None, lse=True, size=1.0):
    rng = np.random.default_rng(seed)
    heads, n = kv * group, len(lengths)
    have = [-(-max(l, 0) // bs) for l in lengths]
    width = max_blocks or max(max(have), 1)
    order_of = rng.permutation(sum(have) + 2)
    pools = Pools(cache, len(order_of), bs, kv, dim, order, pad, seed=seed + 1, size=size)
    table = np.full((n, width + 3), 2 ** 30, np.int64)         # behind what is used: nonsense
    at = 0
    for i, h in enumerate(have):
        h = min(h, width)
        table[i, :h] = order_of[at:at + h]
        at += h
        for j in range(h):
            if rng.random() < bad:
                table[i, j] = rng.choice([-1, len(order_of), -2 ** 31])
    if spoil:
        # whatever is not read is NaN or infinite: places behind a sequence, in front of its window, unused blocks
        seen = np.zeros((len(order_of), bs), bool)
        for i, l in enumerate(lengths):
            l = min(max(l, 0), width * bs)
            for t in range(max(0, l - window) if window else 0, l):
                b = table[i, t // bs]
                if 0 <= b < len(order_of):
                    seen[b, t % bs] = True
        for r, x in zip(pools.raw, (np.nan, np.inf)):
            pools.view(r)[~seen] = R.encode(np.float32(x).reshape(1), cache)[0]
        pools.send()
    q = R.encode((rng.standard_normal((n, heads + 2, dim + q_pad)) * grow).astype(np.float32), kind)
    scale = dim ** -0.5 if scale is None else scale
    d = B.PagedAttentionDesc(pools.layout, kind, n, heads, width, table.shape[1], longest, window, scale, (heads + 2) * (dim + q_pad), dim + q_pad,
                             (heads + 1) * (dim + 8), dim + 8)
    size = q.itemsize
    out = B.DeviceBuffer(n * (heads + 1) * (dim + 8) * size)
    out.fill(0x5A)
    ls = up(np.full(n * heads + 1, 77, np.float32))
    bytes_ = B.ops_paged_attention_workspace(d)
    work = B.DeviceBuffer(bytes_ + 64) if bytes_ else None
    if work:
        work.fill(0xFF)
    args = (d, up(q), *pools.dev, ints(table), ints(lengths), out, ls if lse else None, work)
    ok(B.ops_paged_attention(*args))
    raw = out.to_array(R.np_type(kind)).reshape(n, heads + 1, dim + 8)
    got_lse = ls.to_array()
    ok(B.ops_paged_attention(*args))
    np.testing.assert_array_equal(raw, out.to_array(R.np_type(kind)).reshape(raw.shape))
    got = R.decode(raw, kind)
    sentinel = np.frombuffer(b"\x5a" * size, R.np_type(kind))[0]
    assert (raw[:, heads] == sentinel).all() and (raw[:, :, dim:] == sentinel).all()
    assert got_lse[-1] == 77
    if work:
        assert (work.to_array(np.uint8)[bytes_:] == 0xFF).all()
    qv, kv_, vv = R.decode(q[:, :heads, :dim], kind), pools.values(0), pools.values(1)
    for i, l in enumerate(lengths):
        l = min(max(l, 0), width * bs)
        ts = np.arange(max(0, l - window) if window else 0, l)
        b = table[i, ts // bs] if len(ts) else np.zeros(0, np.int64)
        keep = (b >= 0) & (b < len(order_of))
        b, s = b[keep], ts[keep] % bs
        want, want_lse, tol, tol_lse = R.attend(qv[i], kv_[b, s].transpose(1, 0, 2), vv[b, s].transpose(1, 0, 2), scale)
        # a weight in 16 bits is kept as two terms of its type: 2^-16 of it at most is lost, and for the 16-bit float 2^-24 of the
        # largest at least (its smallest step) a token
        if cache != F32 and kind != F32 and len(b):
            n_seen = len(b)
            tol = tol + (2 * 2.0 ** -16 + (2.0 ** -24 * n_seen if cache == F16 else 0)) * np.abs(vv[b, s]).max()
        err = np.abs(got[i, :heads, :dim] - want)
        lim = tol + HALF[kind] * np.abs(want) + (2.0 ** -25 if kind == F16 else 0)      # (its subnormals' half step)
        assert (err <= lim).all(), (i, l, float((err / np.maximum(lim, 1e-30)).max()))
        if lse:
            g = got_lse[i * heads:(i + 1) * heads]
            assert (np.isneginf(g) == np.isneginf(want_lse)).all()
            fine = np.isfinite(want_lse)
            assert (np.abs(g[fine] - want_lse[fine]) <= tol_lse[fine]).all()
    return got


PAIRS = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]


@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("dim", [8, 16, 32, 40, 64, 72, 80, 96, 112, 128, 136, 192, 248, 256])
def test_attend_head_sizes(kind, cache, dim):
    run_attend(kind, cache, "thd" if dim % 16 else "htd", 16, 2, 3, dim, [1, 200, 0, 77], seed=dim)


@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("group,kv", [(1, 1), (1, 12), (2, 3), (4, 2), (7, 1), (8, 2), (15, 1), (16, 2), (17, 1), (20, 2), (33, 1), (128, 1)])
def test_attend_groups(kind, cache, group, kv):
    run_attend(kind, cache, "thd", 16, kv, group, 64, [130, 1, 33], seed=group)


@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("bs", [1, 2, 3, 4, 8, 16, 24, 32, 33, 64, 128, 1000])
@pytest.mark.parametrize("order", ["thd", "htd"])
def test_attend_block_sizes(kind, cache, bs, order):
    run_attend(kind, cache, order, bs, 2, 4, 64, [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300], seed=bs, pad=8)


@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("longest", [0, 1, 500, 10 ** 9])
def test_attend_long_and_ragged(kind, cache, longest):
    """Long sequences are split, short ones not, whatever the caller expects."""
    run_attend(kind, cache, "thd", 16, 1, 8, 128, [5000, 1, 0, 2047, 2048, 2049, 777, 4096, 511, 512, 513], longest=longest, seed=longest % 97, q_pad=8)


@pytest.mark.parametrize("requests", [63, 64, 65, 255, 256, 257, 1023, 1500])
@pytest.mark.parametrize("window", [0, 700])
def test_attend_many_requests(requests, window):
    """A few long sequences among many short and empty ones."""
    rng = np.random.default_rng(requests)
    lengths = rng.integers(0, 40, requests)
    lengths[rng.integers(0, requests, 6)] = [2500, 1100, 600, 513, 512, 0]
    run_attend(BF16, BF16, "thd", 16, 1, 2, 32, lengths.tolist(), window=window, seed=requests)


@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("requests,kv,group,longest", [(31, 3, 2, 60), (32, 3, 2, 60), (33, 5, 17, 200), (40, 3, 4, 1500), (1, 3, 33, 5000), (290, 3, 1, 700)])
def test_attend_workgroups_by_xcd(kind, cache, requests, kv, group, longest):
    """Heads whose rows end inside lines, several tiles of query heads, shares in all numbers modulo eight."""
    rng = np.random.default_rng(requests)
    lengths = np.exp(rng.uniform(0, np.log(longest), requests)).astype(int)
    lengths[0] = longest
    run_attend(kind, cache, "thd", 16, kv, group, 40, lengths.tolist(), longest=longest, seed=requests)


@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("window", [0, 450])
def test_attend_lengths_around_the_cuts(kind, cache, window):
    """Shares of 128 tokens at most: just below, at and above two, three and more of them, and tiles that they do not divide."""
    run_attend(kind, cache, "thd", 16, 2, 3, 64, [127, 128, 129, 159, 160, 161, 191, 192, 193, 255, 256, 257, 289, 383, 384, 385, 449, 481, 511, 512, 513, 1025, 1153],
               window=window, longest=10 ** 6, seed=window)


@pytest.mark.parametrize("kind,cache,requests,kv,group,dim,longest,rest", [
    (F16, F16, 400, 1, 2, 32, 130000, 3), (F32, BF16, 393, 1, 1, 32, 70001, 200), (BF16, BF16, 49, 8, 2, 40, 4200, 4200), (F32, F32, 130, 3, 2, 64, 5003, 900),
    (BF16, BF16, 100, 4, 1, 256, 4097, 500), (F16, F16, 700, 1, 17, 32, 6000, 60)])
def test_attend_long_ones_in_large_batches(kind, cache, requests, kv, group, dim, longest, rest):
    """Batches that fill the device, whose longest sequence alone is cut into hundreds of shares."""
    rng = np.random.default_rng(longest)
    lengths = np.exp(rng.uniform(0, np.log(rest), requests)).astype(int)
    lengths[requests // 2] = longest
    lengths[-1] = 0
    run_attend(kind, cache, "thd", 16, kv, group, dim, lengths.tolist(), longest=longest, seed=requests)


@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("window", [1, 2, 16, 31, 100, 128, 1000, 10 ** 9])
def test_attend_windows(kind, cache, window):
    run_attend(kind, cache, "htd", 24, 2, 2, 80, [1, 24, 100, 101, 129, 1500, 3001, 0], window=window, seed=window % 89)


@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("bad", [0.1, 0.9, 1.0])
def test_attend_blocks_that_are_not_in_the_pool(kind, cache, bad):
    run_attend(kind, cache, "thd", 4, 2, 2, 64, [1, 24, 100, 333, 3000], bad=bad, seed=3)


@pytest.mark.parametrize("kind,cache", PAIRS)
def test_attend_lengths_beyond_the_row_and_below_zero(kind, cache):
    run_attend(kind, cache, "thd", 16, 2, 2, 64, [100, -1, 64, 65, -2 ** 31], max_blocks=4, seed=9, spoil=False, lse=False)


@pytest.mark.parametrize("kind,cache", PAIRS)
def test_attend_sharp_and_flat_scores(kind, cache):
    run_attend(kind, cache, "thd", 16, 2, 4, 128, [700, 2000], grow=30.0, seed=4)       # one token takes nearly all
    run_attend(kind, cache, "thd", 16, 2, 4, 128, [700, 2000], scale=0.0, seed=5)       # all alike
    run_attend(kind, cache, "thd", 16, 2, 4, 128, [700, 2000], scale=-0.3, seed=6)


@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("group", [1, 2, 4, 8])
def test_attend_small_and_large_values(kind, cache, group):
    """Keys and values that are subnormal in fp16, and ones near its largest; queries far from 1 either way."""
    run_attend(kind, cache, "thd", 16, 2, group, 64, [300, 40], size=2e-6, scale=1000.0, seed=1)
    run_attend(kind, cache, "thd", 16, 2, group, 64, [300, 40], size=12000.0, scale=1e-5, seed=2)
    run_attend(kind, cache, "thd", 16, 2, group, 64, [300, 40], grow=3e-4, scale=300.0, seed=3)
    run_attend(kind, cache, "thd", 16, 2, group, 64, [300, 40], grow=3e3, scale=3e-5, seed=4)


def small_attend(kind, cache, keys, values, q, lengths=None):
    """One request, one block: raw host values [tokens][dim] -> out [heads][dim], lse [heads]."""
    t, dim = keys.shape
    lay = B.CacheLayout(cache, 1, t, 1, dim, t * dim, dim, dim)
    heads = q.shape[0]
    d = B.PagedAttentionDesc(lay, kind, 1, heads, 1, 1, t, 0, 1.0, heads * dim, dim, heads * dim, dim)
    out, ls = B.DeviceBuffer(heads * dim * (4 if kind == F32 else 2)), B.DeviceBuffer(4 * heads)
    n = B.ops_paged_attention_workspace(d)
    ok(B.ops_paged_attention(d, up(R.encode(q, kind)), up(R.encode(keys, cache)), up(R.encode(values, cache)), ints([0]), ints([t if lengths is None else lengths]),
                             out, ls, B.DeviceBuffer(n) if n else None))
    return R.decode(out.to_array(R.np_type(kind)).reshape(heads, dim), kind), ls.to_array()


@pytest.mark.parametrize("kind,cache", PAIRS)
def test_attend_infinite_scores(kind, cache):
    dim, t = 64, 70
    rng = np.random.default_rng(0)
    q = np.ones((2, dim), np.float32)
    keys, values = rng.standard_normal((t, dim)).astype(np.float32), rng.standard_normal((t, dim)).astype(np.float32)
    keys[5:40, 3] = -np.inf                     # -infinity as a score: that token counts nothing
    out, ls = small_attend(kind, cache, keys, values, q)
    keep = np.r_[0:5, 40:t]
    want, want_lse, tol, tol_lse = R.attend(R.decode(R.encode(q, kind), kind), R.decode(R.encode(keys[keep], cache), cache)[None],
                                            R.decode(R.encode(values[keep], cache), cache)[None], 1.0)
    assert (np.abs(out - want) <= tol + 2.0 ** -14 + HALF[kind] * np.abs(want)).all() and (np.abs(ls - want_lse) <= tol_lse).all()
    keys[:, 3] = -np.inf                        # all of them: nothing to attend to
    out, ls = small_attend(kind, cache, keys, values, q)
    assert (out == 0).all() and np.isneginf(ls).all()
    keys[:, 3] = 0
    keys[9, 3] = np.nan                         # a NaN that is seen shows
    out, ls = small_attend(kind, cache, keys, values, q)
    assert np.isnan(out).all() and np.isnan(ls).all()
    keys[9, 3] = 0
    keys[69, 3] = np.inf                        # the formula's infinity - infinity
    out, ls = small_attend(kind, cache, keys, values, q)
    assert np.isnan(out).all()


def test_attend_pool_past_32_bits():
    """Blocks that start behind 2^32 elements and 2^33 bytes."""
    bs, kv, dim, blocks = 16, 8, 128, 264 * 1024
    lay = B.CacheLayout(F16, blocks, bs, kv, dim, bs * kv * dim, kv * dim, dim)
    pools = [B.DeviceBuffer(blocks * bs * kv * dim * 2) for _ in range(2)]
    rng = np.random.default_rng(1)
    pick = np.array([blocks - 1, 131072, 131071, 262144, 0, 262143])
    used = 16 * len(pick) - 3
    rows = rng.standard_normal((used, 2, kv, dim)).astype(np.float16)
    slots = [pick[t // bs] * bs + t % bs for t in range(used)]
    row = 2 * kv * dim
    dev = up(rows)
    ok(B.ops_cache_append(B.CacheAppendDesc(lay, F16, used, row, dim, row, dim), dev.ptr.value, dev.ptr.value + kv * dim * 2, ints(slots), *pools))
    q = rng.standard_normal((1, 16, dim)).astype(np.float16)
    d = B.PagedAttentionDesc(lay, F16, 1, 16, len(pick), len(pick), used, 0, 0.1, 16 * dim, dim, 16 * dim, dim)
    out = B.DeviceBuffer(16 * dim * 2)
    n = B.ops_paged_attention_workspace(d)
    ok(B.ops_paged_attention(d, up(q), *pools, ints(pick), ints([used]), out, None, B.DeviceBuffer(n) if n else None))
    want, _, tol, _ = R.attend(q[0].astype(np.float64), rows[:, 0].transpose(1, 0, 2).astype(np.float64), rows[:, 1].transpose(1, 0, 2).astype(np.float64), 0.1)
    got = out.to_array(np.float16).reshape(16, dim).astype(np.float64)
    assert (np.abs(got - want) <= tol + 2.0 ** -13 + HALF[F16] * np.abs(want)).all()
    # a copy between two far blocks
    t_in = ints(np.broadcast_to(pick, (2, 6)))
    t_out, l_out = ints(np.full((2, 6), -1)), ints([0, 0])
    ok(B.ops_beam_reorder(B.BeamReorderDesc(lay, 2, 2, 6, 6, 6, 1, 0), ints([0, 0]), ints([used, used]), t_in, ints([5, blocks - 2]), t_out, l_out, *pools))
    assert t_out.to_array(np.int32)[6:].tolist() == pick[:5].tolist() + [blocks - 2]
    ok(B.ops_paged_attention(d, up(q), *pools, ints(t_out.to_array(np.int32)[6:]), ints([used]), out, None, B.DeviceBuffer(n) if n else None))
    np.testing.assert_array_equal(out.to_array(np.float16).reshape(16, dim).astype(np.float64), got)
    for p in pools:
        p.free()


# ---- beam search --------------------------------------------------------------------------------
def run_select(kind, requests, beams, logits, n, scores=None, ended=None, end_token=2, pad=0):
    rows, vocab = logits.shape
    rng = np.random.default_rng(rows)
    scores = (-rng.random(rows) * 5).astype(np.float32) if scores is None else np.asarray(scores, np.float32)
    wide = np.full((rows, vocab + pad), np.float32(50), np.float32)
    wide[:, :vocab] = logits
    raw = R.encode(wide, kind)
    d = B.BeamSelectDesc(kind, requests, beams, vocab, n, end_token, vocab + pad)
    best, parents, tokens = (up(np.full(requests * n + 1, -9, t)) for t in (np.float32, np.int32, np.int32))
    bytes_ = B.ops_beam_select_workspace(d)
    work = B.DeviceBuffer(bytes_ + 64) if bytes_ else None
    if work:
        work.fill(0xFF)
    args = (d, up(raw), up(scores), None if ended is None else up(np.asarray(ended, np.uint8)), best, parents, tokens, work)
    for _ in range(2):
        ok(B.ops_beam_select(*args))
    got = [best.to_array(np.float32), parents.to_array(np.int32), tokens.to_array(np.int32)]
    assert all(g[-1] == -9 for g in got)
    if work:
        assert (work.to_array(np.uint8)[bytes_:] == 0xFF).all()
    got = [g[:-1].reshape(requests, n) for g in got]
    want = R.select(R.decode(raw[:, :vocab], kind), scores.astype(np.float64), ended, beams, n, end_token)
    np.testing.assert_array_equal(got[1], want[1])
    np.testing.assert_array_equal(got[2], want[2])
    fine = np.isfinite(want[0])
    assert (np.isneginf(got[0]) == np.isneginf(want[0])).all()
    # the sum of the exponentials in 32 bits a piece of a row (at most 512 terms, each off by its argument's rounding and a few steps, which
    # counts as much as the term does), in 64 above: within 2^-17 of it; then one rounding to 32 bits
    assert (np.abs(got[0][fine] - want[0][fine]) <= 2.0 ** -17 + HALF[F32] * np.abs(want[0][fine])).all()
    return got


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("requests,beams,vocab,n", [(1, 1, 1, 1), (1, 1, 7, 7), (2, 3, 5, 15), (1, 4, 1000, 8), (3, 2, 511, 4), (2, 2, 512, 4), (2, 2, 513, 5),
                                                    (1, 8, 30522, 16), (5, 5, 4097, 1), (2, 1, 70001, 128), (1, 128, 300, 128), (2, 16, 8193, 64), (2, 16, 500, 32),
                                                    (1, 64, 1100, 128), (3, 128, 40, 128), (1, 90, 40000, 10)])
@pytest.mark.parametrize("pad", [0, 1])
def test_select(kind, requests, beams, vocab, n, pad):
    """Values that no two rows share, but 16-bit types make ties inside rows."""
    rng = np.random.default_rng(vocab * 7 + n)
    run_select(kind, requests, beams, rng.standard_normal((requests * beams, vocab)).astype(np.float32) * 3, n, pad=pad)


@pytest.mark.parametrize("kind", [F32, F16, BF16])
def test_select_ties(kind):
    rng = np.random.default_rng(2)
    flat = np.zeros((8, 3001), np.float32)
    run_select(kind, 2, 4, flat, 64, scores=np.zeros(8))                       # all alike: lowest beam, lowest token
    run_select(kind, 2, 4, flat, 64, scores=[0, -1, 0, -1, -2, -2, -2, -2])
    few = rng.integers(0, 3, (8, 5003)).astype(np.float32)                     # thousands of equal values around the border
    run_select(kind, 2, 4, few, 128, scores=-np.arange(8) / 7)
    up_ = np.tile(np.arange(9001, dtype=np.float32) / 900, (2, 1))             # sorted, either way
    run_select(kind, 1, 2, up_, 32, scores=[0, -0.25])
    run_select(kind, 1, 2, up_[:, ::-1].copy(), 32, scores=[0, -0.25])
    zeros = np.where(rng.random((4, 2000)) < 0.5, 0.0, -0.0).astype(np.float32)
    run_select(kind, 1, 4, zeros, 20, scores=[-1, -1, -1, -1])                 # +0 and -0 are equal


@pytest.mark.parametrize("kind", [F32, F16, BF16])
def test_select_masked_logits(kind):
    rng = np.random.default_rng(8)
    x = rng.standard_normal((6, 4001)).astype(np.float32)
    x[:, 50:] = -np.inf
    run_select(kind, 2, 3, x, 64)
    x[:, 3:] = -np.inf                         # fewer allowed tokens than are asked for: the rest at -infinity, lowest first
    run_select(kind, 2, 3, x, 64)
    x[1] = -np.inf                             # a beam without any
    run_select(kind, 2, 3, x, 64)
    x[:] = -np.inf
    run_select(kind, 2, 3, x, 64)
    y = rng.standard_normal((6, 4001)).astype(np.float32)
    y[0, 17], y[2, 4000], y[3, 5], y[4, :] = np.nan, np.inf, -np.inf, np.nan
    run_select(kind, 2, 3, y, 100)
    lowest = np.full((4, 1000), {F32: -3.4e38, F16: -65504.0, BF16: -3.38e38}[kind], np.float32)     # masks of the type's lowest value
    lowest[:, 500] = 1.0
    run_select(kind, 1, 4, lowest, 4)


@pytest.mark.parametrize("kind", [F32, F16, BF16])
def test_select_scores_and_ended_beams(kind):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((8, 6007)).astype(np.float32)
    run_select(kind, 2, 4, x, 8, scores=[0, -np.inf, -np.inf, -np.inf] * 2)    # the first step: one beam only
    run_select(kind, 2, 4, x, 8, scores=[np.nan, np.inf, -1, -2] * 2)
    run_select(kind, 2, 4, x, 8, scores=[-np.inf] * 8)
    run_select(kind, 2, 4, x, 8, ended=[0, 1, 0, 0, 1, 1, 1, 1])
    run_select(kind, 2, 4, x, 16, ended=[1] * 8, scores=[-1, -2, -2, -np.inf, 0, 1, 2, 3])
    run_select(kind, 2, 4, x, 16, ended=[1] * 8, end_token=-1)                 # no token to offer
    run_select(kind, 2, 4, x, 16, ended=[0, 1] * 4, end_token=6006)
    run_select(kind, 2, 4, x, 16, ended=[0, 1] * 4, end_token=6007)
    run_select(kind, 2, 4, x, 8, scores=[-1e30, -5, -1e8, -4] * 2)
    run_select(kind, 2, 4, x, 40, scores=[-1e30, -1e30, -2e30, -3e38] * 2)     # so large that every token offers the same
    run_select(kind, 2, 4, x, 8, scores=[3e38, 1e20, 3e38, -1] * 2)
    x[1] = np.nan                                                              # an ended beam's logits are not read
    run_select(kind, 2, 4, x, 8, ended=[0, 1, 0, 0, 0, 0, 0, 0])


# ---- tables that follow the beams -----------------------------------------------------------------
@pytest.mark.parametrize("cache", [F32, F16, BF16])
@pytest.mark.parametrize("order,bs,kv,dim,rows,table_rows,layers", [("thd", 16, 2, 64, 4, 4, 1), ("htd", 24, 3, 80, 9, 6, 3), ("thd", 1, 1, 8, 5, 5, 2),
                                                                    ("htd", 128, 1, 256, 3, 8, 2), ("thd", 5, 12, 64, 33, 33, 1)])
def test_reorder(cache, order, bs, kv, dim, rows, table_rows, layers):
    rng = np.random.default_rng(rows)
    width = 6
    used = table_rows * width
    numbers = rng.permutation(used + rows + 3)
    pools = Pools(cache, len(numbers), bs, kv, dim, order, 8, layers=layers)
    table = np.full((table_rows, width + 2), -3, np.int64)
    table[:, :width] = numbers[:used].reshape(table_rows, width)
    lengths = rng.integers(0, width * bs + 1, table_rows)
    lengths[0] = width * bs                                   # full
    lengths[1] = bs                                           # ends with a block
    lengths[2] = 0
    parents = rng.integers(0, table_rows, rows)
    parents[0] = 0
    parents[-1] = table_rows                                  # not a row
    parents[1] = -1
    if rows > 3:
        parents[3] = 3
    spare = numbers[used:used + rows].copy()
    if rows > 4:
        parents[4] = 3
        lengths[3] = bs * 2 + min(3, bs - 1)
        if rows > 8:
            spare[8], parents[8] = len(numbers), 3            # not a block
    d = B.BeamReorderDesc(pools.layout, rows, table_rows, width, width + 2, width + 1, layers, pools.per_layer)
    t_out, l_out = ints(np.full(rows * (width + 1), -9)), ints(np.full(rows, -9))
    for _ in range(2):
        ok(B.ops_beam_reorder(d, ints(parents), ints(lengths), ints(table), ints(spare), t_out, l_out, *pools.dev))
    want_t, want_l, want = np.full((rows, width + 1), -9), np.full(rows, -9), [r.copy() for r in pools.raw]
    for i, p in enumerate(parents):
        if not 0 <= p < table_rows:
            continue
        n = lengths[p]
        want_l[i] = n
        full, rest = divmod(int(n), bs)
        want_t[i, :full] = table[p, :full]
        if rest and p == i:
            want_t[i, full] = table[p, full]
        elif rest:
            inside = 0 <= spare[i] < len(numbers)
            want_t[i, full] = spare[i] if inside else -1
            for layer in range(layers if inside else 0):
                for w in want:
                    v = pools.view(w, layer)
                    v[spare[i], :rest] = v[table[p, full], :rest]
    np.testing.assert_array_equal(t_out.to_array(np.int32).reshape(rows, width + 1), want_t)
    np.testing.assert_array_equal(l_out.to_array(np.int32), want_l)
    for g, w in zip(pools.fetch(), want):
        np.testing.assert_array_equal(g, w)


def test_reorder_lengths_and_sources_out_of_range():
    pools = Pools(F16, 12, 4, 1, 16)
    table = np.array([[0, 1, 99], [2, -1, 3], [4, 5, 6]])
    d = B.BeamReorderDesc(pools.layout, 3, 3, 3, 3, 3, 1, 0)
    t_out, l_out = ints(np.full(9, -9)), ints([-9] * 3)
    ok(B.ops_beam_reorder(d, ints([2, 0, 1]), ints([10, 6, 100]), ints(table), ints([9, 10, 11]), t_out, l_out, *pools.dev))
    # row 0 takes row 2 (held to 12 tokens: full), row 1 takes row 0 whose last block is none, row 2 row 1 likewise
    assert t_out.to_array(np.int32).reshape(3, 3).tolist() == [[4, 5, 6], [0, 1, -1], [2, -1, -9]]
    assert l_out.to_array(np.int32).tolist() == [12, 10, 6]
    for g, w in zip(pools.fetch(), pools.raw):
        np.testing.assert_array_equal(g, w)


# ---- together ---------------------------------------------------------------------------------------
def hip(name, *args):
    f = getattr(B.lib(), name)
    f.restype = ctypes.c_int
    assert f(*args) == 0, name


@pytest.mark.parametrize("kind,cache", [(F32, F32), (F32, F16), (BF16, BF16)])
@pytest.mark.parametrize("captured", [False, True])
def test_beam_search_over_a_paged_cache(kind, cache, captured):
    """Prompts, then steps of beam search: plan, append, attend, select, reorder, each on what the one before left on the device, against
    rows of plain arrays.  Captured: a step's calls are recorded into a graph once, with the sizes of the largest step, and replayed."""
    rng = np.random.default_rng(12)
    requests, beams, kv, group, dim, bs, vocab, steps = 3, 4, 2, 3, 32, 8, 701, 12
    rows, heads, width = requests * beams, 6, 12
    blocks = rows * width * 3
    pools = Pools(cache, blocks, bs, kv, dim)
    prompt = [13, 1, 24]
    stream = ctypes.c_void_p()
    hip("hipStreamCreateWithFlags", ctypes.byref(stream), 1)
    L = B.lib()

    free = list(rng.permutation(blocks))
    table = [ints(np.full((rows, width), -1)) for _ in range(2)]
    lengths = ints(np.zeros(rows))
    lengths_next = ints(np.zeros(rows))
    max_tokens = 160
    starts, slots, counts = ints(np.zeros(rows + 1)), ints(np.zeros(max_tokens)), ints(np.zeros(3))
    added, free_dev, spare = ints(np.zeros(rows)), ints(np.zeros(256)), ints(np.zeros(rows))
    size = 4 if kind == F32 else 2
    kv_rows = B.DeviceBuffer(max_tokens * 2 * kv * dim * size)
    q, out = B.DeviceBuffer(rows * heads * dim * size), B.DeviceBuffer(rows * heads * dim * size)
    logits = B.DeviceBuffer(rows * vocab * size)
    scores, best = up(np.zeros(rows, np.float32)), up(np.zeros((requests, beams), np.float32))
    parents, tokens = ints(np.zeros((requests, beams))), ints(np.zeros((requests, beams)))
    plan = B.BlockPlanDesc(rows, blocks, bs, width, width, 256, max_tokens)
    app = B.CacheAppendDesc(pools.layout, kind, max_tokens, 2 * kv * dim, dim, 2 * kv * dim, dim)
    att = B.PagedAttentionDesc(pools.layout, kind, rows, heads, width, width, width * bs, 0, dim ** -0.5, heads * dim, dim, heads * dim, dim)
    sel = B.BeamSelectDesc(kind, requests, beams, vocab, beams, -1, vocab)
    reo = B.BeamReorderDesc(pools.layout, rows, rows, width, width, width, 1, 0)
    work = [B.DeviceBuffer(max(16, n)) for n in (B.ops_paged_attention_workspace(att), B.ops_beam_select_workspace(sel))]

    def put(buf, arr):
        arr = np.ascontiguousarray(arr)
        hip("reef_hal_memcpy_h2d", buf.ptr, arr.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(arr.nbytes))

    def first_half(s):
        ok(B.ops_block_plan(plan, lengths, added, free_dev, table[0], lengths_next, starts, slots, counts, s))
        ok(B.ops_cache_append(app, kv_rows, kv_rows.ptr.value + kv * dim * size, slots, *pools.dev, s))
        ok(B.ops_paged_attention(att, q, *pools.dev, table[0], lengths_next, out, None, work[0], s))

    def second_half(s):
        ok(B.ops_beam_select(sel, logits, scores, None, best, parents, tokens, work[1], s))
        ok(B.ops_beam_reorder(reo, parents, lengths_next, table[0], spare, table[1], lengths, *pools.dev, s))

    graphs = []
    if captured:
        for half in (first_half, second_half):
            graph, run = ctypes.c_void_p(), ctypes.c_void_p()
            hip("hipStreamBeginCapture", stream, 0)
            half(stream)
            hip("hipStreamEndCapture", stream, ctypes.byref(graph))
            hip("hipGraphInstantiate", ctypes.byref(run), graph, None, None, ctypes.c_size_t(0))
            graphs.append((graph, run))

    def do(i):
        if captured:
            hip("hipGraphLaunch", graphs[i][1], stream)
        else:
            (first_half, second_half)[i](stream)
        hip("hipStreamSynchronize", stream)

    rows_of = [[] for _ in range(rows)]          # plain: each row's list of (key, value) rows
    score = np.full(rows, -np.inf, np.float32)
    score[::beams] = 0
    for step in range(steps):
        more = np.ones(rows, int) if step else np.repeat(prompt, beams)
        put(added, more.astype(np.int32))
        put(free_dev, np.array(free[:256], np.int32))
        new = np.zeros((max_tokens, 2, kv, dim), np.float32)
        total = int(more.sum())
        assert total <= max_tokens
        new[:total] = rng.standard_normal((total, 2, kv, dim))
        if not step:                              # a request's beams start alike
            at = np.concatenate([[0], np.cumsum(more)])
            for r in range(rows):
                new[at[r]:at[r + 1]] = new[at[r // beams * beams]:][:more[r]]
        new = R.encode(new, kind)
        put(kv_rows, new)
        qv = R.encode(rng.standard_normal((rows, heads, dim)).astype(np.float32), kind)
        put(q, qv)
        do(0)
        used, tok, bad = counts.to_array(np.int32)
        assert tok == total and bad == 0
        free = free[used:]
        at = 0
        got = R.decode(out.to_array(R.np_type(kind)).reshape(rows, heads, dim), kind)
        for r in range(rows):
            for t in range(at, at + more[r]):
                x = new[t] if kind == cache else R.encode(new[t].astype(np.float32), cache)
                rows_of[r].append(R.decode(x, cache))
            at += more[r]
            have = np.array(rows_of[r])
            want, _, tol, _ = R.attend(R.decode(qv[r], kind), have[:, 0].transpose(1, 0, 2), have[:, 1].transpose(1, 0, 2), dim ** -0.5)
            err = np.abs(got[r] - want)
            assert (err <= tol + 2.0 ** -14 + HALF[kind] * np.abs(want)).all(), (step, r, err.max())
        assert lengths_next.to_array(np.int32).tolist() == [len(x) for x in rows_of]
        lg = R.encode((rng.standard_normal((rows, vocab)) * 2).astype(np.float32), kind)
        put(logits, lg)
        put(scores, score)
        put(spare, np.array(free[-rows:], np.int32))
        do(1)
        want = R.select(R.decode(lg, kind), score.astype(np.float64), None, beams, beams, -1)
        np.testing.assert_array_equal(parents.to_array(np.int32).reshape(requests, beams), want[1])
        np.testing.assert_array_equal(tokens.to_array(np.int32).reshape(requests, beams), want[2])
        score = best.to_array(np.float32).ravel()
        assert np.abs(score - want[0].ravel()).max() <= 2.0 ** -17 + HALF[F32] * np.abs(want[0]).max()
        rows_of = [list(rows_of[p]) for p in want[1].ravel()]
        # who keeps the blocks: whatever the new tables do not name is free again
        t = table[1].to_array(np.int32).reshape(rows, width)
        kept = set(int(t[r, j]) for r in range(rows) for j in range(-(-len(rows_of[r]) // bs)))
        free = [b for b in rng.permutation(blocks) if b not in kept]
        put(table[0], t)
    for graph, run in graphs:
        hip("hipGraphExecDestroy", run)
        hip("hipGraphDestroy", graph)
    hip("hipStreamDestroy", stream)


def test_calls_on_two_streams_do_not_disturb_each_other():
    """Attention and selection side by side, each with a workspace of its own, many times over: the bits of a call alone."""
    rng = np.random.default_rng(1)
    jobs = []
    for s in range(2):
        pools = Pools(BF16, 400, 16, 2, 128, seed=s)
        d = B.PagedAttentionDesc(pools.layout, BF16, 3, 8, 130, 130, 2000, 0, 0.09, 8 * 128, 128, 8 * 128, 128)
        sel = B.BeamSelectDesc(BF16, 2, 3, 9001, 6, -1, 9001)
        stream = ctypes.c_void_p()
        hip("hipStreamCreateWithFlags", ctypes.byref(stream), 1)
        jobs.append(dict(stream=stream, pools=pools, att=d, sel=sel, q=up(R.encode(rng.standard_normal((3, 8, 128)), BF16)),
                         table=ints(rng.integers(0, 400, (3, 130))), lengths=ints([2000, 1, 900]), out=B.DeviceBuffer(3 * 8 * 128 * 2),
                         logits=up(R.encode(rng.standard_normal((6, 9001)), BF16)), scores=up(np.zeros(6, np.float32)), best=B.DeviceBuffer(48),
                         parents=B.DeviceBuffer(48), tokens=B.DeviceBuffer(48), w0=B.DeviceBuffer(max(16, B.ops_paged_attention_workspace(d))),
                         w1=B.DeviceBuffer(max(16, B.ops_beam_select_workspace(sel)))))

    def go(j):
        ok(B.ops_paged_attention(j["att"], j["q"], *j["pools"].dev, j["table"], j["lengths"], j["out"], None, j["w0"], j["stream"]))
        ok(B.ops_beam_select(j["sel"], j["logits"], j["scores"], None, j["best"], j["parents"], j["tokens"], j["w1"], j["stream"]))

    def result(j):
        hip("hipStreamSynchronize", j["stream"])
        return [j[k].to_array(np.uint16) for k in ("out", "best", "parents", "tokens")]

    want = []
    for j in jobs:
        go(j)
        want.append(result(j))
    for _ in range(10):
        for j in jobs:
            j["out"].fill(0)
            j["best"].fill(0)
        B.lib().reef_hal_device_sync()
        for _ in range(20):
            for j in jobs:
                go(j)
        for j, w in zip(jobs, want):
            for a, b in zip(result(j), w):
                np.testing.assert_array_equal(a, b)
    for j in jobs:
        hip("hipStreamDestroy", j["stream"])


# ---- equal and nearly equal offers of different beams ----------------------------------------------
@pytest.mark.parametrize("kind,beams,vocab,n", [(F32, 4, 30522, 8), (F32, 4, 50257, 8), (F16, 20, 30523, 16), (BF16, 4, 128257, 16), (F32, 4, 701, 5),
                                                (BF16, 33, 1001, 32), (F32, 12, 70001, 32)])
def test_select_beams_with_the_same_logits(kind, beams, vocab, n):
    """Beams that hold the same logits and scores offer the same wherever their rows lie: the lowest beam goes first, and neither the choice nor
    a bit of the scores depends on the address of the logits."""
    rng = np.random.default_rng(vocab)
    requests = 3
    one = R.encode((rng.standard_normal((requests, vocab)) * 2.5).astype(np.float32), kind)
    raw = np.repeat(one, beams, axis=0).ravel()
    scores = np.repeat(-rng.random(requests), beams).astype(np.float32)
    x = R.decode(one, kind)
    m = x.max(1, keepdims=True)
    offers = np.repeat(scores[::beams, None].astype(np.float64) + (x - (m + np.log(np.exp(x - m).sum(1, keepdims=True)))), beams, axis=0)
    offers = offers.reshape(requests, beams * vocab)
    at = np.argsort(-offers, axis=1, kind="stable")[:, :n]
    d = B.BeamSelectDesc(kind, requests, beams, vocab, n, -1, vocab)
    first = None
    for ahead in (0, 1, 5, 31):
        dev = up(np.concatenate([np.zeros(ahead, raw.dtype), raw]))
        best, parents, tokens, work = B.DeviceBuffer(4 * requests * n), B.DeviceBuffer(4 * requests * n), B.DeviceBuffer(4 * requests * n), B.DeviceBuffer(
            B.ops_beam_select_workspace(d))
        ok(B.ops_beam_select(d, dev.ptr.value + ahead * raw.itemsize, up(scores), None, best, parents, tokens, work))
        np.testing.assert_array_equal(parents.to_array(np.int32).reshape(requests, n), at // vocab + np.arange(requests)[:, None] * beams)
        np.testing.assert_array_equal(tokens.to_array(np.int32).reshape(requests, n), at % vocab)
        bits = best.to_array(np.uint32)
        first = bits if first is None else first
        np.testing.assert_array_equal(bits, first)


@pytest.mark.parametrize("kind,vocab", [(F32, 30522), (F16, 30523), (BF16, 128257), (F32, 999)])
def test_select_beams_that_differ_in_one_token(kind, vocab):
    """Beams alike but for one unlikely token: their offers lie 1e-9 to 1e-6 apart, and 64 bits tell them apart."""
    rng = np.random.default_rng(vocab)
    x = np.tile((rng.standard_normal(vocab) * 2).astype(np.float32), (8, 1))
    for b, more in enumerate((7, 3, 5, 0, 2, 6, 1, 4)):
        x[b, vocab // 3] = -4 + more / 64
    run_select(kind, 1, 8, x, 24, scores=[-1.0] * 8)
    run_select(kind, 2, 4, x, 10, scores=[-1.0] * 8)


# ---- scores and queries at the ends of their range ---------------------------------------------------
def one_request(kind, cache, keys, values, q, scale):
    """One request, one block: host values [tokens][dim], queries [heads][dim] -> out [heads][dim], lse [heads]."""
    t, dim = keys.shape
    heads = q.shape[0]
    d = B.PagedAttentionDesc(B.CacheLayout(cache, 1, t, 1, dim, t * dim, dim, dim), kind, 1, heads, 1, 1, t, 0, scale, heads * dim, dim, heads * dim, dim)
    out, ls = B.DeviceBuffer(heads * dim * (4 if kind == F32 else 2)), B.DeviceBuffer(4 * heads)
    n = B.ops_paged_attention_workspace(d)
    ok(B.ops_paged_attention(d, up(R.encode(q, kind)), up(R.encode(keys, cache)), up(R.encode(values, cache)), ints([0]), ints([t]), out, ls,
                             B.DeviceBuffer(n) if n else None))
    return R.decode(out.to_array(R.np_type(kind)).reshape(heads, dim), kind), ls.to_array()


@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("tokens", [40, 200, 3000])
@pytest.mark.parametrize("sign", [1, -1])
def test_attend_scores_of_any_size(kind, cache, tokens, sign):
    """Scores from 2^22 to 2^31, where 32 bits keep no fractions: the largest takes everything, two equal ones half each.  One dimension alone
    is not zero and its products are exact, so all other weights are 0 and the two are 1: the result is the mean of two values but for a
    rounding of their sum and of the output.  lse: six roundings to 32 bits, each of at most 2^-24 of a number of its size."""
    rng = np.random.default_rng(tokens)
    dim = 64
    values = rng.standard_normal((tokens, dim)).astype(np.float32)
    v = R.decode(R.encode(values, cache), cache)
    for binade in range(22, 31):
        for more in (1.0, 1.25, 1.5, 1.75):
            keys, q = np.zeros((tokens, dim), np.float32), np.zeros((2, dim), np.float32)
            win = rng.permutation(tokens)[:2]
            # (sign < 0: scores are negative, the largest is the one next to zero)
            keys[:, 5] = 4096 * (rng.integers(1, 5, tokens) / 8 if sign > 0 else 1 + rng.integers(3, 8, tokens) / 8)
            keys[win, 5] = 4096
            q[0, 5], q[1, 5] = sign * 4096 * more, sign * 2048 * more
            out, ls = one_request(kind, cache, keys, values, q, 2.0 ** (binade - 24))
            want = (v[win[0]] + v[win[1]]) / 2
            assert (np.abs(out - want) <= HALF[kind] * np.abs(want) + 2.0 ** -23 * np.abs(v[win]).max(0) + (2.0 ** -25 if kind == F16 else 0)).all(), (binade, more)
            s = np.array([1, 0.5]) * sign * more * 2.0 ** binade
            assert (np.abs(ls - (s + np.log(2))) <= 8 * 2.0 ** -24 * np.abs(s) + 2.0 ** -20).all(), (binade, more)


# ---- the longest sequences ---------------------------------------------------------------------------
@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("group", [1, 4, 20])
def test_attend_windows_of_sequences_just_below_2_31(kind, cache, group):
    """A table whose entries all name one large block holds 2^31 - 2 tokens: places near the end of 32 bits, through all wavefronts."""
    bs, entries, dim = 1549411, 1386, 8
    assert bs * entries == 2 ** 31 - 2
    rng = np.random.default_rng(group)
    raw = [np.zeros((bs, dim), R.np_type(cache)) for _ in range(2)]
    for r in raw:
        r[-6000:] = R.encode(rng.standard_normal((6000, dim)).astype(np.float32), cache)
    k, v = (up(r) for r in raw)
    table = ints(np.zeros(entries))
    q = R.encode(rng.standard_normal((1, group, dim)).astype(np.float32), kind)
    out, ls = B.DeviceBuffer(group * dim * (4 if kind == F32 else 2)), B.DeviceBuffer(4 * group)
    for window in (1, 33, 100, 479, 481, 700, 5000):
        d = B.PagedAttentionDesc(B.CacheLayout(cache, 1, bs, 1, dim, 0, dim, 0), kind, 1, group, entries, entries, 0, window, 0.4, group * dim, dim, group * dim, dim)
        n = B.ops_paged_attention_workspace(d)
        for length in (2 ** 31 - 2, 2 ** 31 - 1, 2 ** 31 - 100):
            held = min(length, bs * entries)
            ok(B.ops_paged_attention(d, up(q), k, v, table, ints([length]), out, ls, B.DeviceBuffer(n) if n else None))
            at = np.arange(held - window, held) % bs
            vv = R.decode(raw[1][at], cache)
            want, want_lse, tol, tol_lse = R.attend(R.decode(q[0], kind), R.decode(raw[0][at], cache)[None], vv[None], 0.4)
            got, got_lse = R.decode(out.to_array(R.np_type(kind)).reshape(group, dim), kind), ls.to_array()
            # (weights of 16-bit types as two terms, as in run_attend)
            extra = (2 * 2.0 ** -16 + (2.0 ** -24 * window if cache == F16 else 0)) * np.abs(vv).max() if cache != F32 and kind != F32 else 0
            assert (np.abs(got - want) <= tol + extra + HALF[kind] * np.abs(want) + (2.0 ** -25 if kind == F16 else 0)).all(), (window, length)
            assert (np.abs(got_lse - want_lse) <= tol_lse).all(), (window, length)


@pytest.mark.parametrize("kind,cache", [(F32, F16), (F32, BF16), (F32, F32)])
def test_attend_queries_far_from_one(kind, cache):
    run_attend(kind, cache, "thd", 16, 2, 4, 64, [300, 40, 2500], grow=1e35, scale=3e-36, seed=1)
    run_attend(kind, cache, "thd", 16, 2, 4, 64, [300, 40, 2500], grow=1e-33, scale=1e32, seed=2)
    if cache == F16:
        # products are made on queries brought near 1, so that nothing between runs over or under either
        run_attend(kind, cache, "thd", 16, 2, 4, 64, [300, 40, 2500], grow=5e37, scale=2e-38, seed=3)
        run_attend(kind, cache, "thd", 16, 2, 4, 64, [300, 40, 2500], grow=1e-37, scale=2e36, seed=4)
        run_attend(kind, cache, "thd", 16, 2, 4, 64, [300, 40, 2500], grow=1e-40, scale=2e38, seed=5)
        rng = np.random.default_rng(6)
        values = rng.standard_normal((50, 64)).astype(np.float32)
        for big in (1e38, 1e-38):
            for scale in (1e6, 2e38):
                out, ls = one_request(kind, cache, np.zeros((50, 64), np.float32), values, np.full((2, 64), big, np.float32), scale)
                want, want_lse, tol, tol_lse = R.attend(np.zeros((2, 64)), np.zeros((1, 50, 64)), R.decode(R.encode(values, cache), cache)[None], 1.0)
                assert (np.abs(out - want) <= tol + HALF[kind] * np.abs(want)).all() and (np.abs(ls - want_lse) <= tol_lse).all()


@pytest.mark.parametrize("kind,cache", [(F32, F16), (F32, BF16), (F32, F32)])
@pytest.mark.parametrize("group", [1, 4, 8])
@pytest.mark.parametrize("grow,scale", [(1e-35, 1e34), (1e-37, 2e36), (1e-38, 2e37), (1e-39, 2e38)])
def test_attend_queries_next_to_nothing(kind, cache, group, grow, scale):
    """Queries that are subnormal, or whose parts in the cache's type would be."""
    run_attend(kind, cache, "thd", 16, 2, group, 64, [300, 40, 2500], grow=grow, scale=scale, seed=4)


def test_attend_small_queries_over_large_keys():
    run_attend(F32, BF16, "thd", 16, 2, 4, 64, [300, 40, 2500], grow=1e-34, size=1e34, scale=0.125, seed=4)


# ---- slots named twice -------------------------------------------------------------------------------
@pytest.mark.parametrize("kind,cache", PAIRS)
def test_append_of_two_tokens_with_one_slot(kind, cache):
    """Whatever 16 bytes of the slot hold belongs to one of the two tokens, in their place; all other slots are as ever."""
    bs, kv, dim, tokens = 16, 3, 72, 600
    rng = np.random.default_rng(0)
    pools = Pools(cache, 64, bs, kv, dim)
    rows = R.encode(rng.standard_normal((tokens, 2, kv, dim)).astype(np.float32), kind)
    slots = rng.permutation(64 * bs)[:tokens]
    twice = rng.permutation(tokens)[:100].reshape(2, 50)
    slots[twice[1]] = slots[twice[0]]
    row = 2 * kv * dim
    dev = up(rows)
    ok(B.ops_cache_append(B.CacheAppendDesc(pools.layout, kind, tokens, row, dim, row, dim), dev.ptr.value, dev.ptr.value + kv * dim * rows.itemsize, ints(slots), *pools.dev))
    cast = rows if kind == cache else R.encode(rows.astype(np.float32), cache)
    per = 16 // cast.itemsize
    for i, got in enumerate(pools.fetch()):
        have, before = pools.view(got).reshape(64 * bs, kv, dim), pools.view(pools.raw[i]).reshape(64 * bs, kv, dim)
        named = set(slots.tolist())
        for s in range(64 * bs):
            if s not in named:
                np.testing.assert_array_equal(have[s], before[s])
                continue
            who = np.flatnonzero(slots == s)
            pieces = have[s].reshape(kv, dim // per, per)
            fits = [(pieces == cast[t, i].reshape(pieces.shape)).all(-1) for t in who]
            assert np.any(fits, axis=0).all()


# ---- tensors -------------------------------------------------------------------------------------------
TENSORS = """
import torch
from reef_amd import binding as B
dev = dict(device="cuda")
ints = lambda *v: torch.tensor(v, dtype=torch.int32, **dev)
lay = B.CacheLayout(2, 10, 16, 2, 64, 2048, 128, 64)
rows = torch.randn(5, 2, 2, 64, **dev).bfloat16()
pools = [torch.zeros(10, 16, 2, 64, dtype=torch.bfloat16, **dev) for _ in range(2)]
app = B.CacheAppendDesc(lay, 2, 5, 256, 64, 256, 64)
slots = ints(3, 159, 16, 0, 40)
"""


def in_a_process(code):
    import os
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", TENSORS + code], capture_output=True, text=True, timeout=600,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0, r.stdout + r.stderr


def test_tensors_of_another_type_or_layout_are_refused():
    in_a_process("""
def no(f, *args):
    try:
        f(*args)
    except TypeError as e:
        assert "operand" in str(e), e
    else:
        raise SystemExit("taken: %s" % (args,))

good = (rows[:, 0], rows[:, 1], slots, *pools)
assert B.ops_cache_append(app, *good) == 0, B.last_error()
assert B.ops_cache_append(app, *good[:3], torch.nn.Parameter(pools[0]), pools[1].untyped_storage()) == 0, B.last_error()
for i, bad in ((2, slots.long()), (2, slots.float()), (2, ints(*range(10))[::2]), (0, rows[:, 0].float()), (1, rows[:, 1].half()), (3, pools[0].float()),
               (0, rows.transpose(-1, -2)), (4, pools[1].cpu())):
    no(B.ops_cache_append, app, *good[:i], bad, *good[i + 1:])
lengths, table = ints(5, 0), torch.zeros(2, 1, dtype=torch.int32, **dev)
q, out, lse = torch.randn(2, 4, 64, **dev).bfloat16(), torch.zeros(2, 4, 64, dtype=torch.bfloat16, **dev), torch.zeros(2, 4, **dev)
att = B.PagedAttentionDesc(lay, 2, 2, 4, 1, 1, 0, 0, 0.125, 256, 64, 256, 64)
good = (q, *pools, table, lengths, out, lse, None)
assert B.ops_paged_attention(att, *good) == 0, B.last_error()
for i, bad in ((4, lengths.long()), (3, table.long()), (6, lse.double()), (6, lse.half()), (5, out.float()), (0, q.float()), (1, pools[0].half()), (4, ints(5, 5, 0, 0)[::2])):
    no(B.ops_paged_attention, att, *good[:i], bad, *good[i + 1:])
wide = B.PagedAttentionDesc(lay, 0, 2, 4, 1, 1, 0, 0, 0.125, 256, 64, 256, 64)
no(B.ops_paged_attention, wide, *good)
assert B.ops_paged_attention(wide, q.float(), *pools, table, lengths, out.float(), lse, None) == 0, B.last_error()
sel = B.BeamSelectDesc(2, 1, 2, 100, 3, 2, 100)
logits, scores, ended = torch.randn(2, 100, **dev).bfloat16(), torch.zeros(2, **dev), torch.tensor([True, False], **dev)
best, parents, tokens = torch.zeros(3, **dev), ints(0, 0, 0), ints(0, 0, 0)
work = torch.empty(B.ops_beam_select_workspace(sel), dtype=torch.uint8, **dev)
for flags in (ended, ended.to(torch.uint8), None):
    assert B.ops_beam_select(sel, logits, scores, flags, best, parents, tokens, work) == 0, B.last_error()
good = (logits, scores, ended, best, parents, tokens, work)
for i, bad in ((0, logits.float()), (1, scores.half()), (2, ended.int()), (4, parents.long()), (5, tokens.float()), (6, work.cpu())):
    no(B.ops_beam_select, sel, *good[:i], bad, *good[i + 1:])
torch.cuda.synchronize()
""")


def test_calls_with_tensors_go_to_the_current_stream_of_torch():
    """Without a stream of their own, behind what torch was given there, and into a graph that torch captures."""
    in_a_process("""
want = [torch.zeros(160, 2, 64, dtype=torch.bfloat16, **dev) for _ in range(2)]
s = torch.cuda.Stream()
big = torch.randn(4096, 4096, **dev)
late = torch.zeros_like(rows)
torch.cuda.synchronize()
with torch.cuda.stream(s):
    for _ in range(30):
        big = big @ big * 1e-4
    late.copy_(rows)
    assert B.ops_cache_append(app, late[:, 0], late[:, 1], slots, *pools) == 0, B.last_error()
s.synchronize()
for i in range(2):
    want[i][slots.long()] = rows[:, i]
    assert torch.equal(pools[i].view(160, 2, 64), want[i])
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    assert B.ops_cache_append(app, late[:, 0], late[:, 1], slots, *pools) == 0, B.last_error()
for step in range(4):
    late.copy_(torch.randn_like(late, dtype=torch.float32).bfloat16())
    slots.copy_(torch.randperm(160, **dev)[:5].int())
    graph.replay()
    torch.cuda.synchronize()
    for i in range(2):
        want[i][slots.long()] = late[:, i]
        assert torch.equal(pools[i].view(160, 2, 64), want[i]), step
""")
