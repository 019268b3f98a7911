"""The operators that serve many requests over a paged cache, on the device against plain forms in 64 bits (tests/serving_ref.py): attention
of new tokens, scores of given tokens, uses of blocks, forks, compaction, and runs of them together."""
import ctypes

import numpy as np
import pytest

from reef_amd import binding as B
from tests import decode_ref as R
from tests import serving_ref as S
from tests.decode_ref import BF16, F16, F32, HALF
from tests.test_gpu_decode_ops import Pools, hip, in_a_process, ints, ok, up

pytestmark = pytest.mark.gpu
PAIRS = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]


def work_of(n):
    """A workspace full of nonsense with some bytes behind it, or none."""
    if not n:
        return None
    w = B.DeviceBuffer(n + 64)
    w.fill(0xFF)
    return w


def behind(w, n):
    assert w is None or (w.to_array(np.uint8)[n:n + 64] == 0xFF).all()


# ---- attention of new tokens --------------------------------------------------------------------
def run_chunk(kind, cache, order, bs, kv, group, dim, cached, added, window=0, pad=0, scale=None, longest=0, seed=0, spoil=True, bad=0.0, q_pad=0, grow=1.0,
              size=1.0, refused=(), extra=5, max_blocks=None, lse=True):
    rng = np.random.default_rng(seed)
    heads, requests = kv * group, len(cached)
    cached, added = np.asarray(cached), np.asarray(added)
    lengths = np.array([c if i in refused else c + a for i, (c, a) in enumerate(zip(cached, added))])
    have = [-(-max(int(n), 0) // bs) for n in lengths]
    width = max_blocks or max(max(have), 1)
    held = lambda n: S.held(n, width, bs)                                                       # noqa: E731
    order_of = rng.permutation(sum(min(h, width) for h in have) + 2)
    pools = Pools(cache, len(order_of), bs, kv, dim, order, pad, seed=seed + 1, size=size)
    table = np.full((requests, width + 3), 2 ** 30, np.int64)
    at = 0
    for i, h in enumerate(have):
        h = min(h, width)
        table[i, :h] = order_of[at:at + h]
        at += h
        for j in range(h):
            if rng.random() < bad:
                table[i, j] = rng.choice([-1, len(order_of), -2 ** 31])
    in_pool = (table >= 0) & (table < len(order_of))
    if spoil:
        # whatever no row sees is NaN or infinite: places behind a sequence, in front of all windows, unused blocks
        seen = np.zeros((len(order_of), bs), bool)
        for i in range(requests):
            n, c = held(lengths[i]), held(cached[i])
            for t in range(max(0, c + 1 - window) if window else 0, n if added[i] and c < n else 0):
                if in_pool[i, t // bs]:
                    seen[table[i, t // bs], t % bs] = True
        for r, x in zip(pools.raw, (np.nan, np.inf)):
            pools.view(r)[~seen] = R.encode(np.float32(x).reshape(1), cache)[0]
        pools.send()
    starts = extra // 2 + np.concatenate([[0], np.cumsum(added)])       # rows in front of the first request, and behind the last
    tokens = int(starts[-1]) + extra - extra // 2
    q = R.encode((rng.standard_normal((tokens, heads + 2, dim + q_pad)) * grow).astype(np.float32), kind)
    scale = dim ** -0.5 if scale is None else scale
    d = B.ChunkAttentionDesc(pools.layout, kind, requests, heads, tokens, width, table.shape[1], longest, window, scale, (heads + 2) * (dim + q_pad), dim + q_pad,
                             (heads + 1) * (dim + 8), dim + 8)
    item = q.itemsize
    out = B.DeviceBuffer(tokens * (heads + 1) * (dim + 8) * item)
    out.fill(0x5A)
    ls = up(np.full(tokens * heads + 1, 77, np.float32))
    n_work = B.ops_chunk_attention_workspace(d)
    work = work_of(n_work)
    args = (d, up(q), *pools.dev, ints(table), ints(starts), ints(cached), ints(lengths), out, ls if lse else None, work)
    ok(B.ops_chunk_attention(*args))
    raw = out.to_array(R.np_type(kind)).reshape(tokens, heads + 1, dim + 8)
    got_lse = ls.to_array()
    ok(B.ops_chunk_attention(*args))
    np.testing.assert_array_equal(raw, out.to_array(R.np_type(kind)).reshape(raw.shape))
    got = R.decode(raw, kind)
    sentinel = np.frombuffer(b"\x5a" * item, R.np_type(kind))[0]
    assert (raw[:, heads] == sentinel).all() and (raw[:, :, dim:] == sentinel).all()
    outside = np.r_[0:starts[0], starts[-1]:tokens]
    assert (raw[outside] == sentinel).all() and got_lse[-1] == 77
    lse_rows = got_lse[:-1].reshape(tokens, heads)
    assert (lse_rows[outside] == 77).all()
    behind(work, n_work)
    qv, kv_, vv = R.decode(q[:, :heads, :dim], kind), pools.values(0), pools.values(1)
    for i in range(requests):
        rows, n = slice(starts[i], starts[i + 1]), held(lengths[i])
        if not added[i]:
            continue
        ts = np.arange(n)
        there = in_pool[i, ts // bs]
        b = np.where(there, table[i, ts // bs], 0)
        want, want_lse, tol, tol_lse = S.chunk(qv[rows], kv_[b, ts % bs].transpose(1, 0, 2), vv[b, ts % bs].transpose(1, 0, 2), held(cached[i]), n, scale, window,
                                               kind, cache, there)
        err = np.abs(got[rows, :heads, :dim] - want)
        lim = tol + HALF[kind] * np.abs(want) + (2.0 ** -25 if kind == F16 else 0)              # (its subnormals' half step)
        assert (err <= lim).all(), (i, int(cached[i]), int(added[i]), float((err / np.maximum(lim, 1e-30)).max()))
        if lse:
            g = lse_rows[rows]
            assert (np.isneginf(g) == np.isneginf(want_lse)).all(), i
            fine = np.isfinite(want_lse)
            assert (np.abs(g[fine] - want_lse[fine]) <= tol_lse[fine]).all(), i
    return got


@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("dim", [8, 16, 32, 40, 64, 72, 80, 96, 104, 128, 136, 160, 192, 200, 248, 256])
def test_chunk_head_sizes(kind, cache, dim):
    run_chunk(kind, cache, "thd" if dim % 16 else "htd", 16, 2, 3, dim, [0, 200, 13, 77], [1, 5, 0, 90], seed=dim)


@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("group,kv", [(1, 1), (1, 12), (2, 3), (3, 5), (4, 2), (7, 1), (8, 2), (16, 2), (17, 1), (33, 1), (128, 1), (200, 1)])
def test_chunk_groups(kind, cache, group, kv):
    run_chunk(kind, cache, "thd", 16, kv, group, 64, [130, 0, 33], [1, 40, 9], seed=group)


@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("bs", [1, 2, 3, 8, 16, 24, 33, 64, 128, 1000])
@pytest.mark.parametrize("order", ["thd", "htd"])
def test_chunk_block_sizes(kind, cache, bs, order):
    run_chunk(kind, cache, order, bs, 2, 2, 64, [0, 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256], [1, 2, 3, 31, 32, 33, 1, 63, 64, 65, 127, 128, 129], seed=bs, pad=8)


@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("longest", [0, 1, 700, 10 ** 9])
@pytest.mark.parametrize("window", [0, 900])
def test_chunk_long_and_ragged(kind, cache, longest, window):
    """Long sequences are split, short ones not, whatever the caller expects; whole prompts, pieces and single tokens."""
    run_chunk(kind, cache, "thd", 16, 1, 4, 128, [4000, 0, 0, 2047, 10, 6000, 511, 0, 1500], [1, 700, 1, 100, 0, 5, 129, 1000, 33], window=window, longest=longest,
              seed=longest % 97, q_pad=8)


@pytest.mark.parametrize("requests", [63, 64, 65, 300, 1500])
@pytest.mark.parametrize("window", [0, 700])
def test_chunk_many_requests(requests, window):
    """A few long sequences and chunks among many short and empty ones."""
    rng = np.random.default_rng(requests)
    cached, added = rng.integers(0, 40, requests), rng.integers(0, 4, requests)
    pick = rng.permutation(requests)[:6]
    cached[pick] = [2500, 1100, 0, 600, 2900, 0]
    added[pick] = [1, 70, 500, 200, 0, 129]
    run_chunk(BF16, BF16, "thd", 16, 1, 2, 32, cached, added, window=window, seed=requests, refused=(int(pick[3]), 5))


@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("window", [1, 2, 31, 64, 100, 1000, 2 ** 31 - 1])
def test_chunk_windows(kind, cache, window):
    run_chunk(kind, cache, "htd", 24, 2, 2, 80, [0, 24, 1000, 129, 0], [200, 100, 150, 1, 1], window=window, seed=window % 89)


@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("bad", [0.1, 0.9, 1.0])
def test_chunk_blocks_that_are_not_in_the_pool(kind, cache, bad):
    run_chunk(kind, cache, "thd", 4, 2, 2, 64, [1, 24, 100, 1500], [3, 150, 1, 40], bad=bad, seed=3)


@pytest.mark.parametrize("kind,cache", PAIRS)
def test_chunk_refused_requests_and_lengths_beyond_the_row(kind, cache):
    run_chunk(kind, cache, "thd", 16, 2, 2, 64, [100, 0, 64, 33], [200, 3, 70, 1], refused=(0, 2, 3), seed=9)
    run_chunk(kind, cache, "thd", 16, 2, 2, 64, [40, -5, 200, 64], [60, 30, 5, 1], max_blocks=4, seed=9, spoil=False, lse=False)


@pytest.mark.parametrize("kind,cache", PAIRS)
def test_chunk_sharp_and_flat_scores(kind, cache):
    run_chunk(kind, cache, "thd", 16, 2, 4, 128, [700, 0], [40, 300], grow=30.0, seed=4)        # one token takes nearly all
    run_chunk(kind, cache, "thd", 16, 2, 4, 128, [700, 0], [40, 300], scale=0.0, seed=5)        # all alike
    run_chunk(kind, cache, "thd", 16, 2, 4, 128, [700, 0], [40, 300], scale=-0.3, seed=6)


@pytest.mark.parametrize("kind,cache", PAIRS)
def test_chunk_small_and_large_values(kind, cache):
    """Keys and values that are subnormal in fp16, and ones near its largest; queries far from 1 either way."""
    for kw in (dict(size=2e-6, scale=1000.0), dict(size=12000.0, scale=1e-5), dict(grow=3e-4, scale=300.0), dict(grow=3e3, scale=3e-5)):
        run_chunk(kind, cache, "thd", 16, 2, 2, 64, [300, 40], [20, 130], seed=1, **kw)


@pytest.mark.parametrize("kind,cache", [(F32, F16), (F32, BF16), (F32, F32)])
def test_chunk_queries_far_from_one(kind, cache):
    for grow, scale in ((1e35, 3e-36), (1e-33, 1e32)) + (((5e37, 2e-38), (1e-37, 2e36), (1e-40, 2e38)) if cache == F16 else ()):
        run_chunk(kind, cache, "thd", 16, 2, 2, 64, [300, 2000], [20, 40], grow=grow, scale=scale, seed=1)


@pytest.mark.parametrize("kind,cache", [(F32, F16), (F32, BF16), (F32, F32)])
@pytest.mark.parametrize("cached,added,window", [([300, 40], [20, 130], 0), ([0, 700, 5], [600, 200, 300], 0), ([1000], [90], 130), ([2000, 50], [5, 1], 0)])
def test_chunk_large_queries_at_full_scale(kind, cache, cached, added, window):
    """Queries of 2^14 and more whose scores are moderate, as keys are small: tiles that all rows see beside ones that some do."""
    for grow, size, scale in ((2e4, 1e-4, 1.0), (7e4, 2e-5, 2.5), (3e4, 5e-5, -1.0)):
        run_chunk(kind, cache, "thd", 16, 2, 2, 64, cached, added, window=window, grow=grow, size=size, scale=scale, seed=1)


def one_request(kind, cache, keys, values, q, scale, cached, longest=0):
    """One request in one block: raw host values keys, values [tokens][dim], q [new][heads][dim] -> out, lse."""
    t, dim = keys.shape
    new, heads = q.shape[:2]
    d = B.ChunkAttentionDesc(B.CacheLayout(cache, 1, t, 1, dim, t * dim, dim, dim), kind, 1, heads, new, 1, 1, longest, 0, scale, heads * dim, dim, heads * dim, dim)
    out, ls = B.DeviceBuffer(new * heads * dim * (4 if kind == F32 else 2)), B.DeviceBuffer(4 * new * heads)
    ok(B.ops_chunk_attention(d, up(R.encode(q, kind)), up(R.encode(keys, cache)), up(R.encode(values, cache)), ints([0]), ints([0, new]), ints([cached]), ints([t]), out, ls,
                             work_of(B.ops_chunk_attention_workspace(d))))
    return R.decode(out.to_array(R.np_type(kind)).reshape(new, heads, dim), kind), ls.to_array().reshape(new, heads)


@pytest.mark.parametrize("cached,new", [(300, 2), (300, 200)])
@pytest.mark.parametrize("size", [1e-30, 1e-33, 1e-36, 1e-38, 1e-40])
def test_chunk_small_32_bit_keys_and_values(cached, new, size):
    """Three numbers of bf16 leave out 2^-134 at most of a key or a value, in fewer bits than 32 below 2^-110: outputs are off by that much more, and by half of the
    smallest 32-bit number; scores by that times the sum of |query|, weights by as much of themselves, twice."""
    rng = np.random.default_rng(new)
    n, dim, left = cached + new, 64, 2.0 ** -134
    small, one = (rng.standard_normal((n, dim)).astype(np.float32) for _ in range(2))
    small *= np.float32(size)
    q = rng.standard_normal((new, 2, dim)).astype(np.float32)
    wide = lambda *a: [x.astype(np.float64) for x in a]                                         # noqa: E731
    qw, sw, ow = wide(q, small, one)
    out, ls = one_request(F32, F32, one, small, q, 0.1, cached)
    want, want_lse, tol, tol_lse = S.chunk(qw, ow[None], sw[None], cached, n, 0.1, 0, F32, F32)
    assert (np.abs(out - want) <= tol + HALF[F32] * np.abs(want) + left + 2.0 ** -150).all()
    assert (np.abs(ls - want_lse) <= tol_lse).all()
    scale = float(np.float32(0.1 / max(size, 1e-37)))
    out, ls = one_request(F32, F32, small, one, q, scale, cached)
    want, want_lse, tol, tol_lse = S.chunk(qw, sw[None], ow[None], cached, n, scale, 0, F32, F32)
    off = left * scale * np.abs(qw).sum(2)
    assert (np.abs(out - want) <= tol + HALF[F32] * np.abs(want) + (2 * off * np.abs(one).max())[:, :, None]).all()
    assert (np.abs(ls - want_lse) <= tol_lse + off).all()


@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("cached,new", [(0, 150), (70, 30), (3000, 140)])
@pytest.mark.parametrize("dim", [40, 64, 128])
def test_chunk_rows_do_not_see_infinities_and_nan_behind_them(kind, cache, cached, new, dim):
    """A key or a value of a later token of the same request is NaN or infinite: rows in front of it are as if it were not there, those from it on show it."""
    rng = np.random.default_rng(cached + dim)
    total = cached + new
    keys, values, q = (rng.standard_normal(s).astype(np.float32) for s in ((total, dim), (total, dim), (new, 2, dim)))
    clean, clean_lse = one_request(kind, cache, keys, values, q, 0.1, cached)
    for what in (np.nan, np.inf, -np.inf):
        for k in (1, new // 2, new - 1):
            at = cached + k
            v2 = values.copy()
            v2[at, 5] = what
            out, ls = one_request(kind, cache, keys, v2, q, 0.1, cached)
            np.testing.assert_array_equal(out[:k], clean[:k])
            assert not np.isfinite(out[k:, :, 5]).any()
            other = np.arange(dim) != 5
            np.testing.assert_array_equal(out[k:, :, other], clean[k:, :, other])
            np.testing.assert_array_equal(ls, clean_lse)
            k2 = keys.copy()
            k2[at, 5] = np.nan
            out, ls = one_request(kind, cache, k2, values, q, 0.1, cached)
            np.testing.assert_array_equal(out[:k], clean[:k])
            assert np.isnan(out[k:]).all() and np.isnan(ls[k:]).all()
            np.testing.assert_array_equal(ls[:k], clean_lse[:k])


@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("tokens", [40, 200, 3000])
@pytest.mark.parametrize("sign", [1, -1])
def test_chunk_scores_of_any_size(kind, cache, tokens, sign):
    """Scores from 2^18 to 2^31: the largest takes everything, two equal ones half each.  One dimension alone is not zero and its
    products are exact, so all other weights are 0 and the two are alike: the result is the mean of two values but for a rounding of their sum and of the output.
    In 16-bit types the two weights w are rounded to the same w (1 + e), |e| up to half a step, while their sum is not: (w (1 + e) a + w (1 + e) b) / (2 w) is the
    mean times 1 + e, so that half a step of the mean is added."""
    rng = np.random.default_rng(tokens)
    dim, new = 64, 3
    values = rng.standard_normal((tokens, dim)).astype(np.float32)
    v = R.decode(R.encode(values, cache), cache)
    for binade in (18, 20, 21, 23, 24, 25, 27, 29, 30):
        for more in (1.0, 1.25, 1.75):
            keys, q = np.zeros((tokens, dim), np.float32), np.zeros((new, 2, dim), np.float32)
            win = rng.permutation(tokens - new)[:2]
            keys[:, 5] = 4096 * (rng.integers(1, 5, tokens) / 8 if sign > 0 else 1 + rng.integers(3, 8, tokens) / 8)
            keys[win, 5] = 4096
            q[:, 0, 5], q[:, 1, 5] = sign * 4096 * more, sign * 2048 * more
            out, ls = one_request(kind, cache, keys, values, q, 2.0 ** (binade - 24), tokens - new)
            want = (v[win[0]] + v[win[1]]) / 2
            half = HALF[kind] * (1 if kind == F32 else 2 + HALF[kind])
            assert (np.abs(out - want) <= half * np.abs(want) + 2.0 ** -22 * np.abs(v[win]).max(0) + (2.0 ** -25 if kind == F16 else 0)).all(), (binade, more)
            s = np.array([1, 0.5]) * sign * more * 2.0 ** binade
            assert (np.abs(ls - (s + np.log(2))) <= 8 * 2.0 ** -24 * np.abs(s) + 2.0 ** -20).all(), (binade, more)


@pytest.mark.parametrize("kind,cache", PAIRS)
def test_chunk_of_sequences_just_below_2_31(kind, cache):
    """A table whose entries all name one large block holds 2^31 - 2 tokens; a window near its end."""
    bs, entries, dim, group, new = 1549411, 1386, 8, 3, 40
    rng = np.random.default_rng(group)
    raw = [np.zeros((bs, dim), R.np_type(cache)) for _ in range(2)]
    for r in raw:
        r[-6000:] = R.encode(rng.standard_normal((6000, dim)).astype(np.float32), cache)
    k, v = (up(r) for r in raw)
    q = R.encode(rng.standard_normal((new, group, dim)).astype(np.float32), kind)
    out, ls = B.DeviceBuffer(new * group * dim * (4 if kind == F32 else 2)), B.DeviceBuffer(4 * new * group)
    for window in (1, 33, 479, 5000):
        d = B.ChunkAttentionDesc(B.CacheLayout(cache, 1, bs, 1, dim, 0, dim, 0), kind, 1, group, new, entries, entries, 0, window, 0.4, group * dim, dim, group * dim, dim)
        held = bs * entries
        ok(B.ops_chunk_attention(d, up(q), k, v, ints(np.zeros(entries)), ints([0, new]), ints([held - new]), ints([2 ** 31 - 1]), out, ls,
                                 work_of(B.ops_chunk_attention_workspace(d))))
        n = window + new - 1
        at = np.arange(held - n, held) % bs
        want, want_lse, tol, tol_lse = S.chunk(R.decode(q, kind), R.decode(raw[0][at], cache)[None], R.decode(raw[1][at], cache)[None], window - 1, n, 0.4, window, kind, cache)
        got, got_lse = R.decode(out.to_array(R.np_type(kind)).reshape(new, group, dim), kind), ls.to_array().reshape(new, group)
        assert (np.abs(got - want) <= tol + HALF[kind] * np.abs(want) + (2.0 ** -25 if kind == F16 else 0)).all(), window
        assert (np.abs(got_lse - want_lse) <= tol_lse).all(), window


@pytest.mark.parametrize("kind,cache,cached,new", [(BF16, BF16, 0, 1500), (F16, F16, 9000, 400), (F32, BF16, 700, 600), (F32, F32, 2000, 300), (BF16, BF16, 30000, 1)])
def test_chunk_large(kind, cache, cached, new):
    run_chunk(kind, cache, "thd", 16, 2, 4, 128, [cached], [new], longest=cached + new, seed=new, extra=0)


@pytest.mark.parametrize("kind,cache", PAIRS)
@pytest.mark.parametrize("cached,added,window", [([15], [1300], 0), ([0, 900], [1100, 700], 0), ([3, 0, 2500, 40], [900, 1, 300, 1000], 1500)])
def test_chunk_prompts_whose_tiles_see_more_and_more(kind, cache, cached, added, window):
    """Few tiles over many tokens: the late ones are cut, the early ones less or not at all."""
    run_chunk(kind, cache, "htd", 64, 1, 2, 64, cached, added, longest=max(c + a for c, a in zip(cached, added)), window=window, seed=len(cached))
    if kind != F32:
        run_chunk(kind, cache, "thd", 16, 1, 1, 104, cached, added, window=window, seed=7)


def test_chunk_many_prompts_and_long_sequences():
    """More than 64 requests, of which some are cut, some in parts, most not."""
    rng = np.random.default_rng(2)
    cached, added = rng.integers(0, 100, 90), rng.integers(1, 40, 90)
    cached[[3, 50, 77, 80]], added[[3, 50, 77, 80]] = [0, 4000, 700, 0], [1200, 100, 900, 0]
    for longest in (0, 4100, 50):
        run_chunk(BF16, BF16, "thd", 16, 1, 2, 64, cached, added, longest=longest, seed=3)
    run_chunk(F32, F16, "thd", 16, 2, 1, 128, cached, added, longest=4100, seed=4, refused=(77, 5))


def test_pools_past_32_bits():
    """Blocks that start behind 2^32 elements and 2^33 bytes: attention, a fork into one, a compaction out of them."""
    bs, kv, dim, blocks = 16, 8, 128, 264 * 1024
    lay = B.CacheLayout(F16, blocks, bs, kv, dim, bs * kv * dim, kv * dim, dim)
    pools = [B.DeviceBuffer(blocks * bs * kv * dim * 2) for _ in range(2)]
    rng = np.random.default_rng(1)
    pick = np.array([blocks - 1, 131072, 131071, 262144, 0, 262143])
    used = 16 * len(pick) - 3
    rows = rng.standard_normal((used, 2, kv, dim)).astype(np.float16)
    slots = [pick[t // bs] * bs + t % bs for t in range(used)]
    dev, row = up(rows), 2 * kv * dim
    ok(B.ops_cache_append(B.CacheAppendDesc(lay, F16, used, row, dim, row, dim), dev.ptr.value, dev.ptr.value + kv * dim * 2, ints(slots), *pools))

    def attend(table, new):
        q = rng.standard_normal((new, 16, dim)).astype(np.float16)
        d = B.ChunkAttentionDesc(lay, F16, 1, 16, new, len(pick), len(pick), used, 0, 0.1, 16 * dim, dim, 16 * dim, dim)
        out = B.DeviceBuffer(new * 16 * dim * 2)
        ok(B.ops_chunk_attention(d, up(q), *pools, table, ints([0, new]), ints([used - new]), ints([used]), out, None, work_of(B.ops_chunk_attention_workspace(d))))
        want, _, tol, _ = S.chunk(q.astype(np.float64), rows[:, 0].transpose(1, 0, 2).astype(np.float64), rows[:, 1].transpose(1, 0, 2).astype(np.float64), used - new, used, 0.1, 0,
                                  F16, F16)
        got = out.to_array(np.float16).reshape(new, 16, dim).astype(np.float64)
        assert (np.abs(got - want) <= tol + HALF[F16] * np.abs(want) + 2.0 ** -25).all()

    attend(ints(pick), 3)
    attend(ints(pick), 70)
    table, lengths, counts = ints(np.stack([pick, np.full(6, -1)])), ints([used, 0]), ints([0, 0])
    ok(B.ops_cache_fork(B.CacheForkDesc(lay, 1, 2, 6, 6, 1, 1, 0), ints([0]), ints([1]), ints([used]), ints([blocks - 2]), table, lengths, counts, *pools))
    assert table.to_array(np.int32)[6:].tolist() == pick[:5].tolist() + [blocks - 2] and counts.to_array(np.int32).tolist() == [1, 0]
    attend(ints(table.to_array(np.int32)[6:]), 3)
    cm = B.CacheCompactDesc(lay, 2, 6, 6, 6, 1, 0)
    packed = ints(np.full((2, 6), -1))
    ok(B.ops_cache_compact(cm, table, lengths, packed, counts, *pools, work_of(B.ops_cache_compact_workspace(cm))))
    assert counts.to_array(np.int32).tolist() == [7, 6] and sorted(set(packed.to_array(np.int32).tolist())) == list(range(7))
    for half in np.split(packed.to_array(np.int32), 2):
        attend(ints(half), 3)


def test_calls_on_two_streams_do_not_disturb_each_other():
    """The calls of two servers side by side, each with workspaces of its own, many times over: the bits of a call alone."""
    rng = np.random.default_rng(1)
    jobs = []
    for s in range(2):
        pools = Pools(BF16, 12000, 16, 2, 64, seed=s)
        att = B.ChunkAttentionDesc(pools.layout, BF16, 3, 8, 420, 260, 260, 4100, 0, 0.12, 8 * 64, 64, 8 * 64, 64)
        sc, sw = B.TokenScoresDesc(BF16, 3, 128257, 20, 128257), B.BlockSweepDesc(3, 12000, 16, 260, 260)
        stream = ctypes.c_void_p()
        hip("hipStreamCreateWithFlags", ctypes.byref(stream), 1)
        jobs.append(dict(stream=stream, pools=pools, att=att, sc=sc, sw=sw, q=up(R.encode(rng.standard_normal((420, 8, 64)), BF16)), table=ints(rng.permutation(12000)[:780]),
                         starts=ints([0, 300, 301, 420]), cached=ints([700, 4000, 0]), lengths=ints([1000, 4001, 119]), out=B.DeviceBuffer(420 * 8 * 64 * 2),
                         logits=up(R.encode(rng.standard_normal((3, 128257)), BF16)), tokens=ints([5, 60000, -1]), scores=B.DeviceBuffer(12), ranks=B.DeviceBuffer(12),
                         entropy=B.DeviceBuffer(12), top=B.DeviceBuffer(240), tops=B.DeviceBuffer(240), uses=B.DeviceBuffer(48000), free=ints(np.zeros(12000)), counts=B.DeviceBuffer(12),
                         w=[work_of(n) for n in (B.ops_chunk_attention_workspace(att), B.ops_token_scores_workspace(sc), B.ops_block_sweep_workspace(sw))]))

    def go(j):
        ok(B.ops_chunk_attention(j["att"], j["q"], *j["pools"].dev, j["table"], j["starts"], j["cached"], j["lengths"], j["out"], None, j["w"][0], j["stream"]))
        ok(B.ops_token_scores(j["sc"], j["logits"], j["tokens"], j["scores"], j["ranks"], j["entropy"], j["top"], j["tops"], j["w"][1], j["stream"]))
        ok(B.ops_block_sweep(j["sw"], j["table"], j["lengths"], j["uses"], j["free"], j["counts"], j["w"][2], j["stream"]))

    def result(j):
        hip("hipStreamSynchronize", j["stream"])
        return [j[k].to_array(np.uint16) for k in ("out", "scores", "ranks", "entropy", "top", "tops", "uses", "free", "counts")]

    assert all(w is not None for j in jobs for w in j["w"])
    want = []
    for j in jobs:
        go(j)
        want.append(result(j))
    for _ in range(8):
        for j in jobs:
            for k in ("out", "scores", "top"):
                j[k].fill(0)
        B.lib().reef_hal_device_sync()
        for _ in range(15):
            for j in jobs:
                go(j)
        for j, w in zip(jobs, want):
            for a, b in zip(result(j), w):
                np.testing.assert_array_equal(a, b)
    for j in jobs:
        hip("hipStreamDestroy", j["stream"])


SERVING = """
heads, top, V = 4, 5, 1000
table, starts, cached, lengths = ints(3, 1, 7, 9).view(2, 2), ints(0, 2, 5), ints(20, 0), ints(22, 3)
pools = [torch.randn(10, 16, 2, 64, **dev).bfloat16() for _ in range(2)]
q, out, lse = torch.randn(5, heads, 64, **dev).bfloat16(), torch.zeros(5, heads, 64, dtype=torch.bfloat16, **dev), torch.zeros(5, heads, **dev)
att = B.ChunkAttentionDesc(lay, 2, 2, heads, 5, 2, 2, 0, 0, 0.125, 256, 64, 256, 64)
attend = [q, *pools, table, starts, cached, lengths, out, lse, None]
sc = B.TokenScoresDesc(2, 3, V, top, V)
logits, tokens = torch.randn(3, V, **dev).bfloat16(), ints(1, 2, 999)
scores, ranks, entropy, best, bests = torch.zeros(3, **dev), ints(0, 0, 0), torch.zeros(3, **dev), ints(*[0] * 15), torch.zeros(15, **dev)
score = [logits, tokens, scores, ranks, entropy, best, bests, None]
sw = B.BlockSweepDesc(2, 10, 16, 2, 2)
uses, free, counts = ints(*[0] * 10), ints(*[0] * 10), ints(0, 0, 0)
sweep = [table, lengths, uses, free, counts, None]
fk = B.CacheForkDesc(lay, 1, 2, 2, 2, 2, 1, 0)
fork = [ints(0), ints(1), ints(18), ints(5, 6), table.clone(), lengths.clone(), ints(0, 0), *pools]
cm = B.CacheCompactDesc(lay, 2, 2, 2, 2, 1, 0)
compact = [table, lengths, torch.zeros_like(table), ints(0, 0), *pools, torch.empty(B.ops_cache_compact_workspace(cm), dtype=torch.uint8, **dev)]

def plain_attention():
    want = torch.zeros(5, heads, 64)
    k, v = ([p[table[i].long()].reshape(32, 2, 64).float().cpu().repeat_interleave(2, 1) for i in range(2)] for p in pools)
    for i in range(2):
        for n, r in enumerate(range(int(starts[i]), int(starts[i + 1]))):
            e = int(cached[i]) + n + 1
            for h in range(heads):
                w = (k[i][:e, h] @ q[r, h].float().cpu() * 0.125).softmax(0)
                want[r, h] = w @ v[i][:e, h]
    return want
"""


def test_tensors_of_another_type_or_layout_are_refused():
    in_a_process(SERVING + """
def no(f, *args):
    try:
        f(*args)
    except TypeError as e:
        assert "operand" in str(e), e
    else:
        raise SystemExit("taken: %s" % (args,))

wide = torch.zeros(2, 4, dtype=torch.int32, **dev)[:, ::2]
for f, d, good, bads in ((B.ops_chunk_attention, att, attend, ((0, q.float()), (0, q.half()), (1, pools[0].half()), (2, pools[1].cpu()), (3, table.long()), (4, starts.float()), (5, cached.long()),
                                                               (6, ints(0, 0, 0, 0)[::2]), (7, out.float()), (8, lse.half()))),
                         (B.ops_token_scores, sc, score, ((0, logits.float()), (1, tokens.long()), (2, scores.double()), (3, ranks.float()), (4, entropy.half()), (5, best.long()),
                                                          (6, bests.double()))),
                         (B.ops_block_sweep, sw, sweep, ((0, table.long()), (0, wide), (1, lengths.float()), (2, uses.long()), (3, free.float()), (4, counts.cpu()))),
                         (B.ops_cache_fork, fk, fork, ((0, ints(0).long()), (3, ints(5, 6).float()), (4, table.long()), (6, ints(0, 0).long()), (7, pools[0].half()), (8, pools[1].cpu()))),
                         (B.ops_cache_compact, cm, compact, ((0, table.long()), (2, table.float()), (3, ints(0, 0).long()), (4, pools[0].float())))):
    assert f(d, *good) == 0, B.last_error()
    for i, bad in bads:
        no(f, d, *good[:i], bad, *good[i + 1:])
""")


def test_calls_with_tensors_go_to_the_current_stream_of_torch():
    """Behind what torch was given there, and into a graph that torch captures, replayed between other work."""
    in_a_process(SERVING + """
def check(step):
    torch.cuda.synchronize()
    want = plain_attention()
    assert (out.float().cpu() - want).abs().max() <= 0.02 * (1 + want.abs().max()), step
    x = logits.double().log_softmax(1)
    assert (scores.double() - x.gather(1, tokens.long()[:, None])[:, 0]).abs().max() <= 1e-4, step
    assert (bests.view(3, top)[:, 1:] <= bests.view(3, top)[:, :-1]).all(), step
    assert (bests.view(3, top).double() - x.topk(top).values).abs().max() <= 1e-4, step
    assert uses.tolist() == [sum(int(b) == n for row, l in zip(table.tolist(), lengths.tolist()) for b in row[:-(-l // 16)]) for n in range(10)], step
    assert counts[2] == 0 and free[:int(counts[0])].tolist() == [n for n in range(10) if uses[n] == 0], step

def calls():
    assert B.ops_chunk_attention(att, *attend) == 0, B.last_error()
    assert B.ops_token_scores(sc, *score) == 0, B.last_error()
    assert B.ops_block_sweep(sw, *sweep) == 0, B.last_error()

s = torch.cuda.Stream()
big, late_q, late_x = torch.randn(4096, 4096, **dev), torch.randn_like(q.float()).bfloat16(), torch.randn(3, V, **dev).bfloat16()
torch.cuda.synchronize()
with torch.cuda.stream(s):
    for _ in range(30):
        big = big @ big * 1e-4
    q.copy_(late_q)
    logits.copy_(late_x)
    calls()
check("stream")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    calls()
for step in range(4):
    q.copy_(torch.randn(5, heads, 64, **dev))
    logits.copy_(torch.randn(3, V, **dev) * 3)
    tokens.copy_(torch.randint(0, V, (3,), **dev))
    table.copy_(torch.randperm(10, **dev)[:4].view(2, 2))
    cached.copy_(ints(step * 7, 28 - step))
    lengths.copy_(cached + ints(2, 3))
    graph.replay()
    check(step)
""")


def test_chunk_of_single_tokens_is_paged_attention():
    """One new token a request: what the operator for single tokens gives, within the roundings of both."""
    rng = np.random.default_rng(3)
    kv, group, dim, bs, lengths = 2, 4, 64, 16, [1, 40, 333, 2000]
    heads, n, width = kv * group, len(lengths), 125
    pools = Pools(BF16, n * width, bs, kv, dim)
    table = rng.permutation(n * width).reshape(n, width)
    q = R.encode(rng.standard_normal((n, heads, dim)).astype(np.float32), BF16)
    out = [B.DeviceBuffer(n * heads * dim * 2) for _ in range(2)]
    ls = [B.DeviceBuffer(n * heads * 4) for _ in range(2)]
    d0 = B.PagedAttentionDesc(pools.layout, BF16, n, heads, width, width, 2000, 0, 0.125, heads * dim, dim, heads * dim, dim)
    d1 = B.ChunkAttentionDesc(pools.layout, BF16, n, heads, n, width, width, 2000, 0, 0.125, heads * dim, dim, heads * dim, dim)
    ok(B.ops_paged_attention(d0, up(q), *pools.dev, ints(table), ints(lengths), out[0], ls[0], work_of(B.ops_paged_attention_workspace(d0))))
    ok(B.ops_chunk_attention(d1, up(q), *pools.dev, ints(table), ints(range(n + 1)), ints(np.array(lengths) - 1), ints(lengths), out[1], ls[1],
                             work_of(B.ops_chunk_attention_workspace(d1))))
    a, b = (R.decode(x.to_array(np.uint16), BF16) for x in out)
    v = np.abs(pools.values(1)).max()
    assert (np.abs(a - b) <= 3 * HALF[BF16] * v).all()
    assert np.abs(ls[0].to_array() - ls[1].to_array()).max() <= 2.0 ** -15


@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("cached,new,group,dim", [(20, 1, 2, 64), (30, 1, 4, 128), (60, 3, 2, 32), (45, 5, 1, 72), (40, 3, 8, 256), (25, 2, 3, 192), (9000, 2, 3, 192)])
def test_chunk_of_few_rows_keeps_its_weights(kind, cached, new, group, dim):
    """Up to 32 rows a request a weight is two numbers of the 16-bit type, which leave out 2^-16 (bf16) or 2^-22 (fp16) of it at most, as in the operator for single
    tokens: the output is off by that times the mean |value|, by fp16's smallest numbers (2^-25 where the largest weight is 2^5), by what 32 bits
    round, and by half its own step."""
    rng = np.random.default_rng(dim)
    n = cached + new
    keys, values, q = (R.decode(R.encode(rng.standard_normal(s).astype(np.float32), kind), kind) for s in ((n, dim), (n, dim), (new, group, dim)))
    scale = 0.1 * dim ** -0.5
    got, lse = one_request(kind, kind, keys.astype(np.float32), values.astype(np.float32), q.astype(np.float32), scale, cached)
    want, want_lse, tol, tol_lse = S.chunk(q, keys[None], values[None], cached, n, scale, 0, kind, kind)
    mean = S.chunk(q, keys[None], np.abs(values)[None], cached, n, scale, 0, kind, kind)[0]
    lim = tol - HALF[kind] * mean + (2.0 ** -16 if kind == BF16 else 2.0 ** -21) * mean + HALF[kind] * np.abs(want) + (2.0 ** -25 if kind == F16 else 0)
    assert (np.abs(got - want) <= lim).all(), float((np.abs(got - want) / lim).max())
    assert (np.abs(lse - want_lse) <= tol_lse).all()


def test_chunk_starts_that_do_not_ascend_stay_inside():
    """Nothing is read or written behind the tensors, whatever starts, cached and lengths hold."""
    rng = np.random.default_rng(1)
    pools = Pools(BF16, 40, 16, 2, 64)
    tokens, heads, n = 50, 4, 5
    q = up(R.encode(rng.standard_normal((tokens, heads, 64)).astype(np.float32), BF16))
    out = up(np.full(tokens * heads * 64 + 64, 0x4242, np.uint16))
    d = B.ChunkAttentionDesc(pools.layout, BF16, n, heads, tokens, 8, 8, 0, 0, 0.125, heads * 64, 64, heads * 64, 64)
    work = work_of(B.ops_chunk_attention_workspace(d))
    for starts in ([0, 50, 0, 50, 0, 50], [-2 ** 31, 2 ** 31 - 1, 3, -7, 60, 2 ** 31 - 1], [50, 40, 30, 20, 10, 0]):
        for lengths in ([128] * 5, [2 ** 31 - 1, -5, 0, 64, 10]):
            ok(B.ops_chunk_attention(d, q, *pools.dev, ints(rng.integers(-3, 50, (n, 8))), ints(starts), ints(rng.integers(-5, 200, n)), ints(lengths), out, None, work))
    assert (out.to_array(np.uint16)[tokens * heads * 64:] == 0x4242).all()
    behind(work, B.ops_chunk_attention_workspace(d))


@pytest.mark.parametrize("kind,cache", [(BF16, BF16), (F32, F16)])
@pytest.mark.parametrize("requests,tokens,dim", [(5, 50, 64), (5, 700, 64), (90, 300, 32), (90, 3000, 128), (1, 400, 64), (3, 20, 192)])
@pytest.mark.parametrize("longest", [0, 3000])
def test_chunk_starts_that_do_not_ascend_stay_inside_where_tiles_are_cut(kind, cache, requests, tokens, dim, longest):
    """The same with tables of some thousand tokens, whose tiles are cut into shares, few and many requests, tiles of both sizes."""
    rng = np.random.default_rng(tokens)
    kv, group, width = 1, 4, 400
    heads, size = kv * group, 4 if kind == F32 else 2
    pools = Pools(cache, 40, 16, kv, dim)
    q = up(R.encode(rng.standard_normal((tokens, heads, dim)).astype(np.float32), kind))
    n = tokens * heads * dim * size // 2
    out, ls = up(np.full(n + 64, 0x4242, np.uint16)), up(np.full(tokens * heads + 16, 77, np.float32))
    d = B.ChunkAttentionDesc(pools.layout, kind, requests, heads, tokens, width, width, longest, 0, 0.125, heads * dim, dim, heads * dim, dim)
    n_work = B.ops_chunk_attention_workspace(d)
    assert n_work
    work = work_of(n_work)
    table = ints(rng.integers(-3, 50, (requests, width)))
    for starts in (np.arange(requests + 1) % 2 * tokens, rng.integers(-2 ** 31, 2 ** 31, requests + 1), np.linspace(tokens, 0, requests + 1), np.zeros(requests + 1), np.full(requests + 1, tokens),
                   np.r_[0, rng.integers(0, tokens + 1, requests)]):
        for lengths in (np.full(requests, 6400), rng.integers(-5, 7000, requests), np.full(requests, 2 ** 31 - 1)):
            for cached in (rng.integers(-5, 6400, requests), np.zeros(requests)):
                ok(B.ops_chunk_attention(d, q, *pools.dev, table, ints(np.asarray(starts, np.int64)), ints(np.asarray(cached, np.int64)), ints(lengths), out, ls, work))
    assert (out.to_array(np.uint16)[n:] == 0x4242).all() and (ls.to_array()[tokens * heads:] == 77).all()
    behind(work, n_work)
    # and a call as it should be in the same workspace afterwards
    fine = np.linspace(0, tokens, requests + 1).astype(np.int64)
    ok(B.ops_chunk_attention(d, q, *pools.dev, table, ints(fine), ints(np.zeros(requests)), ints(fine[1:] - fine[:-1]), out, ls, work))
    got = out.to_array(np.uint16)[:n].copy()
    ok(B.ops_chunk_attention(d, q, *pools.dev, table, ints(fine), ints(np.zeros(requests)), ints(fine[1:] - fine[:-1]), out, ls, work_of(n_work)))
    np.testing.assert_array_equal(got, out.to_array(np.uint16)[:n])


# ---- scores of given tokens ----------------------------------------------------------------------
def run_scores(kind, logits, tokens, top, pad=0, raw=None):
    rows, vocab = logits.shape
    if raw is None:
        raw = R.encode(np.pad(np.asarray(logits, np.float32), ((0, 0), (0, pad)), constant_values=60), kind)
    d = B.TokenScoresDesc(kind, rows, vocab, top, vocab + pad)
    outs = [up(np.full(n + 1, -9, t)) for n, t in ((rows, np.float32), (rows, np.int32), (rows, np.float32), (rows * top, np.int32), (rows * top, np.float32))]
    n_work = B.ops_token_scores_workspace(d)
    work = work_of(n_work)
    args = (d, up(raw), ints(tokens), *outs, work)
    ok(B.ops_token_scores(*args))
    got = [o.to_array(t) for o, t in zip(outs, (np.float32, np.int32, np.float32, np.int32, np.float32))]
    ok(B.ops_token_scores(*args))
    for g, o in zip(got, outs):
        np.testing.assert_array_equal(g, o.to_array(g.dtype))
        assert g[-1] == -9
    behind(work, n_work)
    want = S.scores(R.decode(raw[:, :vocab], kind), np.asarray(tokens), top)
    np.testing.assert_array_equal(got[1][:-1], want[1])
    np.testing.assert_array_equal(got[3][:-1].reshape(rows, top), want[3])
    # an exponential in 32 bits is off by 2^-23 of itself and three roundings of its argument, 2^-22 (1 + |x - m|) in all; the sum of them weighs that by
    # e, and e (1 + |x - m|) / S adds up to at most 2 + log vocab, as an entropy does; sums are in 64 bits.  The entropy's products have the same error again, times |x - m|
    bound = 2.0 ** -22 * (2 + np.log(vocab))
    x = R.decode(raw[:, :vocab], kind)
    x = np.where(np.isnan(x), -np.inf, x)
    with np.errstate(all="ignore"):
        y = x - x.max(1)[:, None]
        e = np.exp(y)
        second = np.where(e > 0, e * (1 + np.abs(y)) * np.abs(y), 0).sum(1) / e.sum(1)
    for g, w, more in ((got[0][:-1], want[0], 0), (got[2][:-1], want[2], 2.0 ** -21 * np.where(np.isfinite(second), second, 0)),
                       (got[4][:-1].reshape(rows, top), want[4], 0)):
        with np.errstate(over="ignore"):
            w = np.where(np.isinf(w.astype(np.float32)), w.astype(np.float32), w)       # (differences that 32 bits do not hold)
        fine = np.isfinite(w)
        assert (np.isfinite(g) == fine).all() and (np.isnan(g) == np.isnan(w)).all()
        lim = np.broadcast_to(bound + more if w.ndim == 1 else bound, w.shape) + HALF[F32] * np.abs(np.where(fine, w, 0))
        assert (np.abs(g - w)[fine] <= lim[fine]).all(), float((np.abs(g - w)[fine] / lim[fine]).max())


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 7), (3, 256), (2, 511), (2, 513), (5, 1000), (1, 30522), (17, 4097), (300, 1025), (2, 70001), (1, 200003)])
def test_scores_sizes(kind, rows, vocab):
    rng = np.random.default_rng(vocab)
    for top in sorted({0, 1, min(5, vocab), min(20, vocab), min(128, vocab)}):
        tokens = rng.integers(0, vocab, rows)
        tokens[-1] = rng.choice([0, vocab - 1, -1, vocab, 2 ** 31 - 1, -2 ** 31])
        run_scores(kind, rng.standard_normal((rows, vocab)) * 2.5, tokens, top, pad=int(rng.integers(0, 4)))


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("rows", [200, 400, 600])
@pytest.mark.parametrize("vocab", [130, 1999, 6001, 20011])
def test_scores_many_rows(kind, rows, vocab):
    """Rows of few and of many units, taken by many wavefronts and by few; some of them masked in front, behind, all over."""
    rng = np.random.default_rng(rows + vocab)
    x = rng.standard_normal((rows, vocab)).astype(np.float32) * 3
    x[1, :vocab // 2], x[2, vocab // 3:], x[3], x[4, 5:] = -np.inf, -np.inf, -np.inf, np.finfo(np.float16).min
    run_scores(kind, x, rng.integers(-1, vocab + 1, rows), 33, pad=int(vocab % 2))


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [300, 9001, 66000])
def test_scores_odd_values(kind, vocab):
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((14, vocab)) * 3
    x[0] = 1.5                                   # all alike
    x[1] = rng.integers(0, 3, vocab)             # many alike
    x[2] = -np.inf                               # nothing
    x[3, :] = -np.inf
    x[3, vocab // 2] = 4.0                       # one token alone
    x[4, rng.permutation(vocab)[:vocab // 2]] = -np.inf
    x[5, [3, vocab - 2]] = np.nan
    x[6, 11] = np.inf
    x[7] = np.nan
    x[8] = np.arange(vocab) * (10000.0 / vocab)  # ascending: the best are last
    x[9] = -np.arange(vocab) * (10000.0 / vocab)
    x[10] = np.where(np.arange(vocab) % 2, 0.0, -0.0)
    x[11] = np.finfo(np.float16).min
    x[11, 7] = np.finfo(np.float16).max
    x[12, 5] = 60000.0                           # takes everything
    x[13] = 1e-7 * rng.standard_normal(vocab)
    for top in (1, 20, 128):
        run_scores(kind, x, rng.integers(0, vocab, 14), top)
        run_scores(kind, x, [7, vocab - 1, 5, vocab // 2, 4, 3, 11, 0, vocab - 1, 0, 1, 7, 5, 2], top)


def test_scores_extremes_of_32_bits():
    x = np.full((3, 1000), -3e38)
    x[0, 5], x[1, 5:9], x[2] = 3e38, [1e30, 1e30, -1e30, 2e30], 1e-40
    run_scores(F32, x, [5, 6, 999], 10)


@pytest.mark.parametrize("kind,many", [(F32, (0x7F800001, 0xFF800001, 0x7FBFFFFF)), (F16, (0x7C01, 0xFC01)), (BF16, (0x7F81, 0xFFBF))])
@pytest.mark.parametrize("vocab", [129, 4096, 70001])
def test_scores_signalling_nan(kind, many, vocab):
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((5, vocab)).astype(np.float32) * 3
    raw = R.encode(x, kind).copy()
    for i, share in enumerate((0.0, 0.01, 0.5, 0.99, 1.0)):
        where = rng.random(vocab) < share
        raw.view(np.uint32 if kind == F32 else np.uint16)[i, where] = rng.choice(many, int(where.sum()))
    assert np.isnan(R.decode(raw, kind)[4]).all()
    run_scores(kind, x, rng.integers(0, vocab, 5), 64, raw=raw)
    run_scores(kind, x, [0, vocab - 1, 1, 2, 3], 7, raw=raw)


# (Values near 2^20 / log2 e, where exponentials are taken otherwise; rows that reach there from below and from above.)
@pytest.mark.parametrize("vocab", [1000, 30011, 150001])
def test_scores_of_large_values(vocab):
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((8, vocab)) * 4
    x[0] += 726817
    x[1] -= 726817
    x[2] += 2.0 ** 24
    x[3] -= 1e30
    x[4] += np.linspace(726700, 726900, vocab)
    x[5] -= np.linspace(726700, 726900, vocab)
    x[6] = np.where(rng.random(vocab) < 0.01, x[6], -3.4e38)
    x[7] = np.where(np.arange(vocab) < vocab - 3, -250000.0 - np.arange(vocab) % 3, -np.inf)
    tokens = rng.integers(0, vocab, 8)
    run_scores(F32, x, tokens, 20)
    run_scores(F32, x, [vocab - 1] * 8, 0)


# (Places behind a row's end are filled with -2^18 at most: rows whose largest logit is not far above.)
@pytest.mark.parametrize("rows,vocab", [(7, 5), (7, 301), (7, 1026), (7, 2050), (7, 30011), (2, 150001), (300, 1270), (300, 9001), (600, 515), (600, 7001)])
def test_scores_just_above_what_stands_behind_the_end(rows, vocab):
    rng = np.random.default_rng(vocab)
    above = np.array([0.5, 1.0, 10.0, 30.0, 100.0, 740.0, 2000.0])[np.arange(rows) % 7]
    flat = np.repeat((above - 2.0 ** 18)[:, None], vocab, 1)
    for x in (flat, flat - rng.integers(0, 64, (rows, vocab)) / 8, np.where(rng.random((rows, vocab)) < 0.5, flat, -np.inf)):
        x[:, 0] = flat[:, 0]
        run_scores(F32, x, np.where(np.arange(rows) % 3 == 2, rng.integers(0, vocab, rows), 0), min(vocab, 5))


# ---- blocks ---------------------------------------------------------------------------------------
def run_sweep(table, lengths, blocks, bs, max_blocks):
    rows, stride = table.shape
    d = B.BlockSweepDesc(rows, blocks, bs, max_blocks, stride)
    uses, free, counts = (ints(np.full(n + 1, -7)) for n in (blocks, blocks, 3))
    n_work = B.ops_block_sweep_workspace(d)
    work = work_of(n_work)
    for _ in range(2):
        ok(B.ops_block_sweep(d, ints(table), ints(lengths), uses, free, counts, work))
    want = S.sweep(table, lengths, blocks, bs, max_blocks)
    uses, free, counts = (x.to_array(np.int32) for x in (uses, free, counts))
    np.testing.assert_array_equal(uses[:-1], want[0])
    np.testing.assert_array_equal(free[:len(want[1])], want[1])
    assert (free[len(want[1]):] == -7).all() and uses[-1] == -7 and counts.tolist() == want[2] + [-7]
    behind(work, n_work)


@pytest.mark.parametrize("rows,blocks,bs,max_blocks", [(0, 5, 16, 3), (1, 1, 1, 1), (3, 63, 16, 8), (9, 64, 8, 12), (40, 1025, 16, 20), (100, 8192, 24, 50), (100, 8193, 24, 50),
                                                       (700, 4096, 16, 64), (513, 40000, 32, 70), (3, 5000, 1, 20000), (2, 12289, 7, 11111)])
def test_sweep(rows, blocks, bs, max_blocks):
    rng = np.random.default_rng(blocks)
    for bad in (0.0, 0.2):
        table = rng.integers(0, blocks, (rows, max_blocks + 3))
        table[rng.random(table.shape) < bad] = rng.choice([-1, blocks, 2 ** 31 - 1, -2 ** 31])
        lengths = rng.integers(-5, max_blocks * bs + 10, rows) * (rng.random(rows) < 0.7)
        run_sweep(table, lengths, blocks, bs, max_blocks)


def test_sweep_of_nothing_and_of_all():
    table = np.arange(20000).reshape(20, 1000)[:, ::-1].copy()
    run_sweep(table, np.zeros(20, int), 20000, 4, 1000)
    run_sweep(table, np.full(20, 4000), 20000, 4, 1000)
    run_sweep(table, np.full(20, 2 ** 31 - 1), 20000, 4, 1000)
    run_sweep(np.full((500, 300), 9999), np.full(500, 1200), 10001, 4, 300)      # one block, 150000 times


def moved(pools, moves, bs):
    """The pools on the host after copies of the first tokens of blocks, in all layers."""
    want = [r.copy() for r in pools.raw]
    for layer in range(pools.layers or 1):
        for r, w in zip(pools.raw, want):
            a, b = pools.view(r, layer), pools.view(w, layer)
            for m in moves:
                n = m[2] if len(m) > 2 else bs
                b[m[1], :n] = a[m[0], :n]
    return want


def run_fork(pools, parents, children, tokens, free, table, lengths, max_blocks):
    blocks, bs = pools.shape[:2]
    d = B.CacheForkDesc(pools.layout, len(parents), len(table), max_blocks, table.shape[1], len(free), pools.layers or 1, pools.per_layer)
    t, ls, counts = up(np.concatenate([table.ravel(), [-7]]).astype(np.int32)), ints(list(lengths) + [-7]), ints([-7] * 3)
    args = (d, ints(parents), ints(children), ints(tokens), ints(free) if len(free) else None, t, ls, counts, *pools.dev)
    for _ in range(2):                       # again over its own results: the same
        ok(B.ops_cache_fork(*args))
    want = S.fork(parents, children, tokens, free, table, lengths, blocks, bs, max_blocks)
    np.testing.assert_array_equal(t.to_array(np.int32), np.concatenate([want[0].ravel(), [-7]]))
    np.testing.assert_array_equal(ls.to_array(np.int32), want[1].tolist() + [-7])
    assert counts.to_array(np.int32).tolist() == want[2] + [-7]
    for g, w in zip(pools.fetch(), moved(pools, want[3], bs)):
        np.testing.assert_array_equal(g, w)


@pytest.mark.parametrize("cache,order,bs,kv,dim,layers,forks", [(F32, "thd", 16, 2, 8, 1, 1), (BF16, "htd", 16, 3, 40, 3, 7), (F16, "thd", 1, 1, 64, 2, 20), (F32, "htd", 24, 5, 72, 2, 60),
                                                                (BF16, "thd", 7, 12, 256, 1, 33), (BF16, "thd", 4, 1, 8, 1, 255), (F16, "htd", 4, 2, 8, 2, 1100)])
@pytest.mark.parametrize("pad", [0, 16])
def test_fork(cache, order, bs, kv, dim, layers, forks, pad):
    rng = np.random.default_rng(forks)
    base, max_blocks = 1 + forks // 3, 6
    rows = base + forks
    used = rows * max_blocks
    pools = Pools(cache, used + forks + 3, bs, kv, dim, order, pad, layers)
    numbers = rng.permutation(used + forks + 3)
    table = np.full((rows, max_blocks + 2), -1, np.int64)
    table[:, :max_blocks] = numbers[:used].reshape(rows, max_blocks)
    rows_of = rng.permutation(rows)
    lengths = rng.integers(0, max_blocks * bs + 1, rows)
    parents, children = rng.choice(rows_of[:base], forks), rows_of[base:]
    tokens = rng.integers(0, max_blocks * bs + 5, forks)
    for free in (forks + 3, forks // 2, 0):
        pools.send()
        run_fork(pools, parents, children, tokens, numbers[used:used + free], table, lengths, max_blocks)


def test_fork_odd_rows_and_blocks():
    pools = Pools(F16, 20, 4, 1, 16, layers=2)
    table = np.array([[0, 1, 99], [2, -1, 3], [4, 5, 6], [7, 8, 9], [10, 11, 12], [13, 14, 15], [-4, -4, -4], [-4, -4, -4], [-4, -4, -4], [-4, -4, -4]])
    # parents of more tokens than a row holds, of fewer than none, blocks that are none, rows that are none, its own child
    run_fork(pools, [0, 0, 1, 2, -1, 3, 12, 4], [6, 7, 8, 9, 5, 3, 4, 10], [100, 11, 6, 9, 3, 3, 3, 3], [16, 99, 17, 18], table, [9, 7, 50, 3, 3, 3, 0, 0, 0, 0], 3)
    pools.send()
    run_fork(pools, [0, 1], [6, 7], [-5, 3], [16], table, [-9, 2 ** 31 - 1] + [0] * 8, 3)
    pools.send()
    run_fork(pools, [], [], [], [16], table, [0] * 10, 3)


def run_compact(pools, table, lengths, max_blocks, out_pad=0):
    blocks, bs = pools.shape[:2]
    rows, stride = table.shape
    before = np.full((rows, max_blocks + out_pad), -3)
    d = B.CacheCompactDesc(pools.layout, rows, max_blocks, stride, max_blocks + out_pad, pools.layers or 1, pools.per_layer)
    out, counts = up(np.concatenate([before.ravel(), [-7]]).astype(np.int32)), ints([-7] * 3)
    n_work = B.ops_cache_compact_workspace(d)
    work = work_of(n_work)
    for _ in range(2):                       # from the old table again: the same
        ok(B.ops_cache_compact(d, ints(table), ints(lengths), out, counts, *pools.dev, work))
    want = S.compact(table, lengths, before, blocks, bs, max_blocks)
    np.testing.assert_array_equal(out.to_array(np.int32), np.concatenate([want[0].ravel(), [-7]]))
    assert counts.to_array(np.int32).tolist() == want[1] + [-7]
    for g, w in zip(pools.fetch(), moved(pools, want[2], bs)):
        np.testing.assert_array_equal(g, w)
    behind(work, n_work)
    return want


@pytest.mark.parametrize("cache,order,blocks,bs,kv,dim,layers", [(F32, "thd", 1, 16, 2, 8, 1), (BF16, "htd", 63, 16, 3, 40, 3), (F16, "thd", 500, 1, 1, 64, 2), (F32, "htd", 130, 24, 5, 72, 2),
                                                                 (BF16, "thd", 90, 7, 12, 256, 1), (BF16, "thd", 9000, 2, 1, 8, 1), (F16, "htd", 20000, 1, 2, 8, 2)])
@pytest.mark.parametrize("share", [0.0, 0.05, 0.5, 0.95, 1.0])
def test_compact(cache, order, blocks, bs, kv, dim, layers, share):
    rng = np.random.default_rng(blocks)
    used = int(blocks * share)
    numbers = rng.permutation(blocks)[:used]
    max_blocks = 1 + used // 7
    rows = 8 + (used > 0)
    pools = Pools(cache, blocks, bs, kv, dim, order, 8 if bs > 1 else 0, layers)
    table, lengths, at = np.full((rows, max_blocks + 1), 2 ** 30), np.zeros(rows, int), 0
    for i in range(rows):
        n = min(used - at, max_blocks) if i < 8 else min(3, used, max_blocks)
        table[i, :n] = numbers[at:at + n] if i < 8 else numbers[:n]             # (the last row shares its blocks)
        lengths[i] = max(0, n * bs - int(rng.integers(0, bs)))
        at += n if i < 8 else 0
    run_compact(pools, table, lengths, max_blocks, out_pad=2)


def test_compact_entries_that_are_no_blocks():
    pools = Pools(BF16, 12, 4, 2, 16, layers=2)
    run_compact(pools, np.array([[11, -1, 3], [12, 11, 2 ** 31 - 1], [7, 0, 0]]), [12, 100, -4], 3)
    pools = Pools(BF16, 12, 4, 2, 16)
    run_compact(pools, np.zeros((0, 3), int), [], 3)


# ---- together -------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind,cache", [(F32, F32), (F32, F16), (BF16, BF16)])
@pytest.mark.parametrize("captured", [False, True])
def test_serving_over_a_paged_cache(kind, cache, captured):
    """Prompts in pieces, samples forked from them, single tokens of all, requests that end, a compaction now and then: sweep, fork, plan, append,
    attend, score, compact, each on what the one before left on the device, against rows of plain arrays.  Captured: the calls of a step are
    recorded into graphs once and replayed."""
    rng = np.random.default_rng(5)
    rows, kv, group, dim, bs, vocab, steps = 8, 2, 3, 32, 8, 501, 14
    heads, width, blocks, room, top = kv * group, 12, 150, 112, 4
    pools = Pools(cache, blocks, bs, kv, dim)
    stream = ctypes.c_void_p()
    hip("hipStreamCreateWithFlags", ctypes.byref(stream), 1)
    size = 4 if kind == F32 else 2
    table, table2 = (ints(np.full((rows, width), -1)) for _ in range(2))
    cached, lengths, added = (ints(np.zeros(rows)) for _ in range(3))
    parents, children, prefix = (ints(np.full(rows, -1)) for _ in range(3))
    uses, free, counts, fork_counts, plan_counts = (ints(np.zeros(n)) for n in (blocks, blocks, 3, 2, 3))
    starts, slots = ints(np.zeros(rows + 1)), ints(np.zeros(room))
    kv_rows, q, out = B.DeviceBuffer(room * 2 * kv * dim * size), B.DeviceBuffer(room * heads * dim * size), B.DeviceBuffer(room * heads * dim * size)
    logits, given = B.DeviceBuffer(room * vocab * size), ints(np.zeros(room))
    score, rank, entropy, best, best_score = (B.DeviceBuffer(4 * n) for n in (room, room, room, room * top, room * top))
    sw = B.BlockSweepDesc(rows, blocks, bs, width, width)
    fk = B.CacheForkDesc(pools.layout, rows, rows, width, width, 20, 1, 0)
    plan = B.BlockPlanDesc(rows, blocks, bs, width, width, 40, room)
    app = B.CacheAppendDesc(pools.layout, kind, room, 2 * kv * dim, dim, 2 * kv * dim, dim)
    att = B.ChunkAttentionDesc(pools.layout, kind, rows, heads, room, width, width, width * bs, 0, dim ** -0.5, heads * dim, dim, heads * dim, dim)
    sc = B.TokenScoresDesc(kind, room, vocab, top, vocab)
    cm = B.CacheCompactDesc(pools.layout, rows, width, width, width, 1, 0)
    works = [work_of(n) for n in (B.ops_block_sweep_workspace(sw), B.ops_chunk_attention_workspace(att), B.ops_token_scores_workspace(sc), B.ops_cache_compact_workspace(cm))]

    def put(buf, arr):
        arr = np.ascontiguousarray(arr)
        hip("reef_hal_memcpy_h2d", buf.ptr, arr.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(arr.nbytes))

    def fork(s):
        ok(B.ops_block_sweep(sw, table, cached, uses, free, counts, works[0], s))
        ok(B.ops_cache_fork(fk, parents, children, prefix, free, table, cached, fork_counts, *pools.dev, s))
        ok(B.ops_block_sweep(sw, table, cached, uses, free, counts, works[0], s))

    def step(s):
        ok(B.ops_block_plan(plan, cached, added, free, table, lengths, starts, slots, plan_counts, s))
        ok(B.ops_cache_append(app, kv_rows, kv_rows.ptr.value + kv * dim * size, slots, *pools.dev, s))
        ok(B.ops_chunk_attention(att, q, *pools.dev, table, starts, cached, lengths, out, None, works[1], s))
        ok(B.ops_token_scores(sc, logits, given, score, rank, entropy, best, best_score, works[2], s))

    def compact(s):
        ok(B.ops_cache_compact(cm, table, lengths, table2, counts, *pools.dev, works[3], s))

    calls, graphs = (fork, step, compact), []
    if captured:
        for c in calls:
            graph, run = ctypes.c_void_p(), ctypes.c_void_p()
            hip("hipStreamBeginCapture", stream, 0)
            c(stream)
            hip("hipStreamEndCapture", stream, ctypes.byref(graph))
            hip("hipGraphInstantiate", ctypes.byref(run), graph, None, None, ctypes.c_size_t(0))
            graphs.append((graph, run))

    def do(i):
        if captured:
            hip("hipGraphLaunch", graphs[i][1], stream)
        else:
            calls[i](stream)
        hip("hipStreamSynchronize", stream)

    seqs = [[] for _ in range(rows)]             # plain: each row's list of (key, value) rows
    for number in range(steps):
        # requests that end, samples of others in their place
        par, chi, pre = np.full(rows, -1), np.full(rows, -1), np.zeros(rows, int)
        live = [i for i in range(rows) if seqs[i]]
        if number and live:
            for i in rng.permutation(rows)[:2]:
                p = int(rng.choice(live))
                if p not in chi and i not in par and p != i:
                    seqs[i] = seqs[p][:int(rng.integers(0, len(seqs[p]) + 1))]
                    k = int((chi >= 0).sum())
                    par[k], chi[k], pre[k] = p, i, len(seqs[i])
                    live = [j for j in live if j != i]
        put(parents, par.astype(np.int32))
        put(children, chi.astype(np.int32))
        put(prefix, pre.astype(np.int32))
        do(0)
        assert fork_counts.to_array(np.int32)[1] == (par < 0).sum()
        assert cached.to_array(np.int32).tolist() == [len(x) for x in seqs]
        more = np.array([int(rng.integers(1, 14)) if len(seqs[i]) < 20 else 1 for i in range(rows)]) * (rng.random(rows) < 0.8)
        more = np.minimum(more, [width * bs - len(x) for x in seqs])
        total = int(more.sum())
        assert total <= room
        put(added, more.astype(np.int32))
        new = R.encode(rng.standard_normal((room, 2, kv, dim)).astype(np.float32), kind)
        put(kv_rows, new)
        qv = R.encode(rng.standard_normal((room, heads, dim)).astype(np.float32), kind)
        put(q, qv)
        lg = R.encode((rng.standard_normal((room, vocab)) * 2).astype(np.float32), kind)
        put(logits, lg)
        tok = rng.integers(0, vocab, room).astype(np.int32)
        put(given, tok)
        do(1)
        assert plan_counts.to_array(np.int32)[1:].tolist() == [total, 0]
        got, at = R.decode(out.to_array(R.np_type(kind)).reshape(room, heads, dim), kind), 0
        for i in range(rows):
            first = len(seqs[i])
            for t in range(at, at + more[i]):
                seqs[i].append(R.decode(new[t] if kind == cache else R.encode(new[t].astype(np.float32), cache), cache))
            if more[i]:
                have = np.array(seqs[i])
                want, _, tol, _ = S.chunk(R.decode(qv[at:at + more[i]], kind), have[:, 0].transpose(1, 0, 2), have[:, 1].transpose(1, 0, 2), first, len(have), dim ** -0.5, 0,
                                          kind, cache)
                assert (np.abs(got[at:at + more[i]] - want) <= tol + HALF[kind] * np.abs(want)).all(), (number, i)
            at += more[i]
        want = S.scores(R.decode(lg, kind), tok, top)
        np.testing.assert_array_equal(rank.to_array(np.int32), want[1])
        np.testing.assert_array_equal(best.to_array(np.int32).reshape(room, top), want[3])
        assert np.abs(score.to_array() - want[0]).max() <= 2.0 ** -18 * (1 + np.abs(want[0]).max())
        if number % 3 == 2:
            do(2)
            used, _ = counts.to_array(np.int32)[:2]
            t2 = table2.to_array(np.int32).reshape(rows, width)
            named = {int(t2[i, j]) for i in range(rows) for j in range(-(-len(seqs[i]) // bs))}
            assert named == set(range(used))
            put(table, t2)
        put(cached, np.array([len(x) for x in seqs], np.int32))
    for graph, run in graphs:
        hip("hipGraphExecDestroy", run)
        hip("hipGraphDestroy", graph)
    hip("hipStreamDestroy", stream)
