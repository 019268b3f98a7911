"""The operators that serve many requests over a paged cache, what needs no device: refused calls, and the plain forms against each other.  A
refusal comes before anything is launched, so the addresses here are never followed."""
import ctypes

import numpy as np
import pytest

from reef_amd import binding as B
from tests import decode_ref as R
from tests import serving_ref as S
from tests.test_decode_ops import BAD_LAYOUTS, BF16, F16, F32, P, layout, refused


def call(name, desc, *args):
    return B._op(name)(ctypes.addressof(desc) if desc is not None else None, *args, None)


def chunk(cache, **kw):
    v = dict(type=BF16, requests=2, heads=8, tokens=9, max_blocks=4, table_stride=4, longest=0, window=0, scale=0.125, query_stride=512,
             query_head_stride=64, out_stride=512, out_head_stride=64)
    v.update(kw)
    return B.ChunkAttentionDesc(cache=cache, **v)


def scores(**kw):
    v = dict(type=BF16, rows=3, vocab=1000, top=5, logits_stride=1000)
    v.update(kw)
    return B.TokenScoresDesc(**v)


def sweep(**kw):
    v = dict(rows=3, blocks=100000, block_size=16, max_blocks=4, table_stride=4)
    v.update(kw)
    return B.BlockSweepDesc(**v)


def fork(cache, **kw):
    v = dict(forks=2, table_rows=4, max_blocks=4, table_stride=4, free_blocks=3, layers=1, layer_stride=0)
    v.update(kw)
    return B.CacheForkDesc(cache=cache, **v)


def compact(cache, **kw):
    v = dict(rows=4, max_blocks=4, table_stride=4, out_stride=4, layers=1, layer_stride=0)
    v.update(kw)
    return B.CacheCompactDesc(cache=cache, **v)


def addresses(n, **kw):
    """Far from each other, so that nothing overlaps."""
    a = [P + (i << 40) for i in range(n)]
    for k, v in kw.items():
        a[int(k[1:])] = v
    return a


BIG = 1 << 40


def test_layouts_that_are_refused():
    for change, text in BAD_LAYOUTS:
        c = layout(**change)
        refused(call("chunk_attention", chunk(c, type=c.type), *addresses(10), BIG), text)
        refused(call("cache_fork", fork(c), *addresses(9)), text)
        refused(call("cache_compact", compact(c), *addresses(7), BIG), text)
        with pytest.raises(B.ReefError):
            B.ops_chunk_attention_workspace(chunk(c, type=c.type))
        with pytest.raises(B.ReefError):
            B.ops_cache_compact_workspace(compact(c))


@pytest.mark.parametrize("change,text", [
    (dict(type=F16), "type"), (dict(type=7), "type"), (dict(heads=7), "heads"), (dict(heads=0), "heads"), (dict(requests=-1), "requests"), (dict(tokens=-1), "tokens"),
    (dict(requests=1 << 23, heads=8), "too many"), (dict(tokens=1 << 26, heads=8), "too many"), (dict(max_blocks=0), "table"), (dict(table_stride=3), "table"),
    (dict(max_blocks=1 << 28, table_stride=1 << 28), "table"), (dict(window=-1), "window"), (dict(longest=-5), "length"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(scale=3e38), "scale"), (dict(query_stride=500), "16 bytes"), (dict(query_head_stride=-64), "16 bytes"),
    (dict(out_head_stride=60), "16 bytes"), (dict(out_head_stride=0), "overlap"), (dict(out_stride=448), "overlap"), (dict(out_stride=64, out_head_stride=64), "overlap")])
def test_chunk_refusals(change, text):
    d = chunk(layout(), **change)
    refused(call("chunk_attention", d, *addresses(10), BIG), text)
    with pytest.raises(B.ReefError):
        B.ops_chunk_attention_workspace(d)


def test_chunk_pointers_and_workspace():
    d = chunk(layout(blocks=10000), requests=3, tokens=3000, max_blocks=4000, table_stride=4000)
    for i in range(9):
        for bad in ((None, P + 2) if i != 8 else (P + 2,)):
            refused(call("chunk_attention", d, *addresses(10, **{"a%d" % i: bad}), BIG), "unaligned")
    need = B.ops_chunk_attention_workspace(d)
    if need:
        refused(call("chunk_attention", d, *addresses(10), need - 1), "workspace")
        refused(call("chunk_attention", d, *addresses(10, a9=None), need), "workspace")
        refused(call("chunk_attention", d, *addresses(10, a9=P + 8), need), "workspace")
    refused(call("chunk_attention", None, *addresses(10), BIG), "null")
    for kw in (dict(requests=0), dict(tokens=0)):
        assert call("chunk_attention", chunk(layout(), **kw), *[None] * 10, 0) == 0


def test_chunk_workspace_goes_by_the_descriptor():
    """Not more than a few hundred MB, whatever the sizes, and none for short sequences."""
    assert B.ops_chunk_attention_workspace(chunk(layout(), longest=64)) == 0
    for tokens in (1, 100, 8192, 1 << 18):
        for requests in (1, 60, 3000):
            n = B.ops_chunk_attention_workspace(chunk(layout(blocks=1 << 20), requests=requests, tokens=tokens, max_blocks=1 << 14, table_stride=1 << 14))
            assert 0 <= n < 1 << 30


@pytest.mark.parametrize("kind,cache", [(BF16, BF16), (F16, F16), (F32, F32), (F32, F16)])
@pytest.mark.parametrize("heads,kv,dim", [(64, 8, 128), (32, 8, 128), (128, 8, 128), (64, 64, 64), (16, 1, 256), (256, 128, 96)])
def test_chunk_workspace_holds_shares_of_cut_tiles_alone(kind, cache, heads, kv, dim):
    """Up to 3 workgroups for each that runs at once are cut for, 768 of 256 rows or their like, and a cut tile has two shares at least: 1536 of them, and one or two
    a cache head by rounding, of 256 rows of 128 values and 2 numbers, 4 bytes each; lists of requests and items beside them."""
    c = layout(type=cache, blocks=1 << 20, block_size=16, kv_heads=kv, head_dim=dim, block_stride=16 * kv * dim, slot_stride=kv * dim, head_stride=dim)
    for requests, tokens in ((1, 1 << 15), (4, 1 << 15), (16, 1 << 15), (16, 1 << 16), (64, 1 << 12), (65, 1 << 12), (1000, 3000), (200, 1700)):
        n = B.ops_chunk_attention_workspace(chunk(c, type=kind, requests=requests, tokens=tokens, heads=heads, max_blocks=1 << 12, table_stride=1 << 12,
                                                  query_stride=heads * dim, query_head_stride=dim, out_stride=heads * dim, out_head_stride=dim))
        assert 0 <= n < (1536 + 2 * kv) * 256 * 130 * 4 + (1 << 22), (requests, tokens, n)


@pytest.mark.parametrize("change,text", [(dict(type=3), "type"), (dict(rows=-1), "sizes"), (dict(rows=1 << 24), "sizes"), (dict(vocab=0), "sizes"), (dict(vocab=1 << 24), "sizes"),
                                         (dict(top=-1), "given"), (dict(top=129), "given"), (dict(vocab=4), "given"), (dict(logits_stride=999), "overlap"),
                                         (dict(rows=1 << 20, vocab=1 << 20, logits_stride=1 << 20), "2^40")])
def test_scores_refusals(change, text):
    d = scores(**change)
    refused(call("token_scores", d, *addresses(8), BIG), text)
    with pytest.raises(B.ReefError):
        B.ops_token_scores_workspace(d)


def test_workspaces_of_another_descriptor():
    """Smaller ones would be read behind their end."""
    descs = dict(chunk_attention=chunk(layout()), token_scores=scores(), block_sweep=sweep(), cache_compact=compact(layout()), cache_fork=fork(layout()))
    for name in ("chunk_attention", "token_scores", "block_sweep", "cache_compact"):
        f = getattr(B, "ops_%s_workspace" % name)
        assert f(descs[name]) >= 0
        for other, d in descs.items():
            if ctypes.sizeof(d) != ctypes.sizeof(descs[name]):
                with pytest.raises(TypeError):
                    f(d)
        with pytest.raises(TypeError):
            f(None)


def test_scores_pointers():
    d = scores()
    need = B.ops_token_scores_workspace(d)
    for i in range(7):
        for bad in (None, P + 1):
            refused(call("token_scores", d, *addresses(8, **{"a%d" % i: bad}), BIG), "unaligned")
    if need:
        refused(call("token_scores", d, *addresses(8), need - 1), "workspace")
        refused(call("token_scores", d, *addresses(8, a7=P + 8), need), "workspace")
    a = addresses(8)
    refused(call("token_scores", d, *addresses(8, a2=a[0] + 64), BIG), "overlaps")
    refused(call("token_scores", d, *addresses(8, a3=a[1] + 8), BIG), "overlaps")
    refused(call("token_scores", None, *a, BIG), "null")
    assert call("token_scores", scores(rows=0), *[None] * 8, 0) == 0


TABLES = [(dict(rows=-1), "rows"), (dict(rows=1 << 24), "rows"), (dict(blocks=0), "pool"), (dict(block_size=0), "pool"), (dict(blocks=1 << 28), "pool"), (dict(max_blocks=0), "table"),
          (dict(table_stride=3), "table"), (dict(max_blocks=1 << 28, table_stride=1 << 28), "table")]


@pytest.mark.parametrize("change,text", TABLES)
def test_sweep_refusals(change, text):
    d = sweep(**change)
    refused(call("block_sweep", d, *addresses(6), BIG), text)
    with pytest.raises(B.ReefError):
        B.ops_block_sweep_workspace(d)


def test_sweep_pointers():
    d = sweep()
    need = B.ops_block_sweep_workspace(d)
    assert need > 0 and B.ops_block_sweep_workspace(sweep(blocks=100)) == 0
    for i in range(5):
        for bad in (None, P + 2):
            refused(call("block_sweep", d, *addresses(6, **{"a%d" % i: bad}), BIG), "unaligned")
    refused(call("block_sweep", d, *addresses(6), need - 1), "workspace")
    refused(call("block_sweep", d, *addresses(6, a5=None), need), "workspace")
    refused(call("block_sweep", d, *addresses(6, a3=addresses(6)[0]), need), "overlaps")
    refused(call("block_sweep", None, *addresses(6), need), "null")


@pytest.mark.parametrize("change,text", [(dict(forks=-1), "forks"), (dict(forks=5), "forks"), (dict(forks=32769, table_rows=40000), "forks"), (dict(free_blocks=-1), "free"), (dict(layers=0), "layers"), (dict(layers=30001), "layers"),
                                         (dict(layers=2, layer_stride=64), "overlap"), (dict(table_rows=-1), "rows"), (dict(max_blocks=0), "table"), (dict(table_stride=3), "table")])
def test_fork_refusals(change, text):
    refused(call("cache_fork", fork(layout(), **change), *addresses(9)), text)


def test_fork_pointers():
    d = fork(layout())
    for i in range(9):
        for bad in (None, P + (2 if i < 7 else 8)):
            refused(call("cache_fork", d, *addresses(9, **{"a%d" % i: bad})), "unaligned")
    a = addresses(9)
    refused(call("cache_fork", d, *addresses(9, a0=a[4])), "overlaps")
    refused(call("cache_fork", d, *addresses(9, a3=a[5])), "overlaps")
    refused(call("cache_fork", None, *a), "null")
    big = layout(blocks=1, block_size=1 << 24, block_stride=0, kv_heads=2, head_dim=64, slot_stride=128)
    refused(call("cache_fork", fork(big), *a), "too large")


@pytest.mark.parametrize("change,text", [(dict(layers=0), "layers"), (dict(layers=2, layer_stride=64), "overlap"), (dict(rows=-1), "rows"), (dict(max_blocks=0), "table"),
                                         (dict(table_stride=3), "table"), (dict(out_stride=3), "table")])
def test_compact_refusals(change, text):
    d = compact(layout(), **change)
    refused(call("cache_compact", d, *addresses(7), BIG), text)
    with pytest.raises(B.ReefError):
        B.ops_cache_compact_workspace(d)


def test_compact_pointers():
    d = compact(layout())
    need = B.ops_cache_compact_workspace(d)
    for i in range(6):
        for bad in (None, P + (2 if i < 4 else 8)):
            refused(call("cache_compact", d, *addresses(7, **{"a%d" % i: bad}), BIG), "unaligned")
    refused(call("cache_compact", d, *addresses(7), need - 1), "workspace")
    refused(call("cache_compact", d, *addresses(7, a6=P + 8), need), "workspace")
    refused(call("cache_compact", d, *addresses(7, a2=addresses(7)[0]), need), "overlaps")
    refused(call("cache_compact", None, *addresses(7), need), "null")


def test_descriptors_of_other_calls_are_refused():
    with pytest.raises(TypeError):
        B.ops_block_sweep(scores(), *[P] * 5)
    with pytest.raises(TypeError):
        B.ops_cache_fork(fork(layout()), *[P] * 8)


def test_the_plain_form_of_chunks_is_that_of_single_tokens():
    rng = np.random.default_rng(0)
    kv, heads, n, dim = 2, 6, 40, 16
    k, v, q = rng.standard_normal((kv, n, dim)), rng.standard_normal((kv, n, dim)), rng.standard_normal((5, heads, dim))
    for window in (0, 7):
        out, lse, _, _ = S.chunk(q, k, v, 35, n, 0.3, window, F32, F32)
        for i in range(5):
            at = slice(max(0, 36 + i - window) if window else 0, 36 + i)
            want, want_lse, _, _ = R.attend(q[i], k[:, at], v[:, at], 0.3)
            np.testing.assert_allclose(out[i], want, rtol=1e-12)
            np.testing.assert_allclose(lse[i], want_lse, rtol=1e-12)
