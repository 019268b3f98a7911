"""The operators of text generation, what needs no device: places in a paged cache, and refused calls.  A refusal comes before
anything is launched, so the addresses here are never followed."""
import ctypes

import numpy as np
import pytest

from reef_amd import binding as B

P = 4096        # an aligned address
F32, F16, BF16 = 0, 1, 2


def layout(**kw):
    v = dict(type=BF16, blocks=10, block_size=16, kv_heads=2, head_dim=64, block_stride=2048, slot_stride=128, head_stride=64)
    v.update(kw)
    return B.CacheLayout(**v)


def test_places_of_tokens():
    c = layout()
    row = [3, 9, -1, 10, 0, 2 ** 31 - 1]
    assert B.ops_paged_row(c, row, 0) == 3 * 2048
    assert B.ops_paged_row(c, row, 31) == 9 * 2048 + 15 * 128
    assert B.ops_paged_row(c, row, 64) == 0
    for token in (32, 47, 48, 63, 80, 96, 2 ** 40, -1):     # block -1, block 10 of 10, a wild one, behind the row
        assert B.ops_paged_row(c, row, token) is None


def test_places_past_32_bits():
    c = layout(blocks=2 ** 20, block_size=1024, block_stride=1024 * 2048, slot_stride=2048, head_stride=64)
    assert B.ops_paged_row(c, [2 ** 20 - 1], 1023) == (2 ** 20 - 1) * 1024 * 2048 + 1023 * 2048
    c = layout(block_size=3)
    assert B.ops_paged_row(c, [1, 2], 5) == 2 * 2048 + 2 * 128


def test_places_for_any_block_size():
    """The kernels multiply and shift where this divides."""
    rng = np.random.default_rng(0)
    sizes = list(range(1, 70)) + [2 ** k + j for k in range(7, 16) for j in (-1, 0, 1)] + rng.integers(1, 2 ** 16, 40).tolist()
    row = np.zeros(1 << 14, np.int32)
    for bs in sizes:
        c = layout(blocks=1, block_size=bs, slot_stride=8, head_stride=8, head_dim=8, kv_heads=1, block_stride=0)
        held = min(len(row) * bs, 2 ** 31 - 1)
        for t in [0, 1, bs - 1, bs, bs + 1, 2 * bs - 1, held - 1, held // bs * bs - 1] + rng.integers(0, held, 30).tolist():
            assert B.ops_paged_row(c, row, t) == t % bs * 8, (bs, t)
        if held == len(row) * bs:
            assert B.ops_paged_row(c, row, held) is None
    # quotients: a row whose entries name themselves
    row = np.arange(4096, dtype=np.int32)
    for bs in (1, 3, 7, 16, 24, 100, 1000, 524287, 524288):
        c = layout(blocks=4096, block_size=bs, slot_stride=8, head_stride=8, head_dim=8, kv_heads=1, block_stride=2 ** 40)
        for t in [0, 4095 * bs, min(4096 * bs, 2 ** 31) - 1] + rng.integers(0, min(4096 * bs, 2 ** 31 - 1), 50).tolist():
            assert B.ops_paged_row(c, row, t) == t // bs * 2 ** 40 + t % bs * 8, (bs, t)


BAD_LAYOUTS = [(dict(type=3), "type"), (dict(type=-1), "type"), (dict(blocks=0), "bad cache"), (dict(block_size=0), "bad cache"),
               (dict(kv_heads=0), "bad cache"), (dict(blocks=2 ** 20, block_size=2 ** 11), "bad cache"), (dict(head_dim=60), "head_dim"),
               (dict(head_dim=264), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(head_stride=63), "16 bytes"),
               (dict(head_stride=32), "overlap"), (dict(slot_stride=64), "overlap"), (dict(slot_stride=0), "overlap"),
               (dict(block_stride=1024), "overlap"), (dict(block_stride=-2048), "16 bytes"), (dict(block_stride=2 ** 61), "too large")]


def refused(status, text):
    assert status == 1
    assert text in B.last_error(), B.last_error()


def call(name, desc, *args):
    return B._op(name)(ctypes.addressof(desc), *args, None)


def attention(cache, **kw):
    v = dict(type=BF16, requests=2, heads=8, max_blocks=4, table_stride=4, longest=0, window=0, scale=0.125, query_stride=512,
             query_head_stride=64, out_stride=512, out_head_stride=64)
    v.update(kw)
    return B.PagedAttentionDesc(cache=cache, **v)


def append(cache, **kw):
    v = dict(type=BF16, tokens=3, key_stride=128, key_head_stride=64, value_stride=128, value_head_stride=64)
    v.update(kw)
    return B.CacheAppendDesc(cache=cache, **v)


def reorder(cache, **kw):
    v = dict(rows=4, table_rows=4, max_blocks=4, table_stride=4, out_stride=4, layers=1, layer_stride=0)
    v.update(kw)
    return B.BeamReorderDesc(cache=cache, **v)


def test_layouts_that_are_refused():
    for change, text in BAD_LAYOUTS:
        c = layout(**change)
        refused(B.ops_cache_append(append(c, type=c.type), P, P, P, P, P), text)
        refused(call("paged_attention", attention(c, type=c.type), *[P] * 8, 1 << 40), text)
        refused(B.ops_beam_reorder(reorder(c), P, P, P, P, 2 * P, P, P, P), text)
        with pytest.raises(B.ReefError):
            B.ops_paged_attention_workspace(attention(c, type=c.type))


def test_steps_of_one_place_may_be_anything():
    c = layout(kv_heads=1, head_stride=1, blocks=1, block_stride=0)
    assert B.ops_paged_attention_workspace(attention(c)) >= 0
    c = layout(type=F32, head_dim=8, kv_heads=1, head_stride=0, slot_stride=8, block_stride=128)
    assert B.ops_paged_attention_workspace(attention(c, type=F32)) >= 0


@pytest.mark.parametrize("change,text", [(dict(type=F16), "type"), (dict(type=7), "type"), (dict(tokens=-1), "negative"),
                                         (dict(key_stride=100), "16 bytes"), (dict(value_head_stride=-64), "16 bytes")])
def test_append_refusals(change, text):
    refused(B.ops_cache_append(append(layout(), **change), P, P, P, P, P), text)


def test_append_pointers():
    for i in range(5):
        for bad in (None, P + (2 if i == 2 else 8)):
            args = [P] * 5
            args[i] = bad
            refused(B.ops_cache_append(append(layout()), *args), "unaligned")
    assert B.ops_cache_append(append(layout(), tokens=0), None, None, None, None, None) == 0
    refused(B._op("cache_append")(None, P, P, P, P, P, None), "null")


@pytest.mark.parametrize("change,text", [(dict(type=F16), "type"), (dict(heads=7), "heads"), (dict(heads=0), "heads"), (dict(requests=-1), "requests"),
                                         (dict(requests=1 << 23, heads=8), "too many"), (dict(max_blocks=0), "table"), (dict(table_stride=3), "table"),
                                         (dict(max_blocks=1 << 28, table_stride=1 << 28), "table"), (dict(window=-1), "window"),
                                         (dict(longest=-5), "length"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
                                         (dict(query_stride=500), "16 bytes"), (dict(out_head_stride=60), "16 bytes")])
def test_attention_refusals(change, text):
    d = attention(layout(), **change)
    refused(call("paged_attention", d, *[P] * 8, 1 << 40), text)
    with pytest.raises(B.ReefError):
        B.ops_paged_attention_workspace(d)


def test_attention_pointers_and_workspace():
    d = attention(layout())
    for i in range(7):
        for bad in ((None, P + 2) if i != 6 else (P + 2,)):
            args = [P] * 7
            args[i] = bad
            refused(call("paged_attention", d, *args, P, 1 << 40), "unaligned")
    assert call("paged_attention", attention(layout(), requests=0), *[None] * 8, 0) == 0


@pytest.mark.parametrize("change,text", [(dict(requests=-1), "negative"), (dict(free_blocks=-1), "negative"), (dict(max_tokens=-1), "negative"),
                                         (dict(blocks=0), "pool"), (dict(block_size=0), "pool"), (dict(blocks=1 << 20, block_size=1 << 11), "pool"),
                                         (dict(max_blocks=0), "table"), (dict(table_stride=7), "table"), (dict(max_blocks=1 << 28, table_stride=1 << 28), "table")])
def test_plan_refusals(change, text):
    v = dict(requests=2, blocks=10, block_size=16, max_blocks=8, table_stride=8, free_blocks=4, max_tokens=8)
    v.update(change)
    refused(B.ops_block_plan(B.BlockPlanDesc(**v), *[P] * 8), text)


def test_outputs_over_inputs():
    d = B.BlockPlanDesc(2, 10, 16, 8, 8, 4, 8)
    good = [i * P for i in range(1, 9)]
    for out in range(3, 8):
        for i in range(3):
            args = list(good)
            args[out] = good[i] + 4
            refused(B.ops_block_plan(d, *args), "overlap")
    d = B.BeamSelectDesc(BF16, 2, 4, 100, 8, 2, 100)
    good = [i * P for i in range(1, 8)]
    for out in range(3, 7):
        for i in range(3):
            args = list(good)
            args[out] = good[i] & ~15
            refused(call("beam_select", d, *args, 1 << 40), "overlap")


def test_plan_pointers():
    d = B.BlockPlanDesc(2, 10, 16, 8, 8, 4, 8)
    for i in range(8):
        for bad in (None, P + 1):
            args = [P] * 8
            args[i] = bad
            refused(B.ops_block_plan(d, *args), "unaligned")


@pytest.mark.parametrize("change,text", [(dict(type=5), "type"), (dict(requests=-1), "sizes"), (dict(beams=0), "sizes"), (dict(beams=129), "sizes"),
                                         (dict(vocab=0), "sizes"), (dict(vocab=1 << 24), "sizes"), (dict(requests=1 << 22), "sizes"), (dict(select=0), "select"),
                                         (dict(select=129), "select"), (dict(vocab=2, logits_stride=2, select=9), "select"), (dict(logits_stride=99), "overlap"),
                                         (dict(requests=1 << 18, vocab=1 << 23, logits_stride=1 << 23), "2^40")])
def test_select_refusals(change, text):
    v = dict(type=F32, requests=2, beams=4, vocab=100, select=8, end_token=2, logits_stride=100)
    v.update(change)
    d = B.BeamSelectDesc(**v)
    refused(call("beam_select", d, *[P] * 7, 1 << 40), text)
    with pytest.raises(B.ReefError):
        B.ops_beam_select_workspace(d)


def test_select_pointers():
    d = B.BeamSelectDesc(BF16, 2, 4, 100, 8, 2, 100)
    for i in (0, 1, 3, 4, 5):
        for bad in (None, P + 1):
            args = [P] * 6
            args[i] = bad
            refused(call("beam_select", d, *args, P, 1 << 40), "unaligned")


@pytest.mark.parametrize("change,text", [(dict(rows=-1), "rows"), (dict(table_rows=0), "rows"), (dict(layers=0), "layers"), (dict(max_blocks=0), "table"),
                                         (dict(out_stride=3), "table"), (dict(table_stride=3), "table"), (dict(layers=2, layer_stride=2048), "overlap"),
                                         (dict(layers=2, layer_stride=20484), "16 bytes")])
def test_reorder_refusals(change, text):
    refused(B.ops_beam_reorder(reorder(layout(), **change), P, P, P, P, 2 * P, P, P, P), text)


def test_reorder_of_huge_blocks():
    c = layout(block_size=1 << 23, slot_stride=128, block_stride=1 << 30)
    refused(B.ops_beam_reorder(reorder(c, max_blocks=1, table_stride=1, out_stride=1), P, P, P, P, 2 * P, 3 * P, P, P), "too large")


def test_reorder_pointers():
    d = reorder(layout(), layers=2, layer_stride=20480)
    good = [P, P, P, P, 2 * P, 3 * P, P, P]
    for i in range(8):
        for bad in (None, good[i] + 2):
            args = list(good)
            args[i] = bad
            refused(B.ops_beam_reorder(d, *args), "unaligned")
    refused(B.ops_beam_reorder(d, P, P, P, P, P, 3 * P, P, P), "overlap")
    refused(B.ops_beam_reorder(d, P, P, P, P, P + 60, 3 * P, P, P), "overlap")
    refused(B.ops_beam_reorder(d, P, P, P, P, 2 * P, P + 12, P, P), "overlap")


def test_tensors_of_a_torch_that_came_later_are_refused():
    """Loaded first, the library has a HIP runtime of its own; in a process of its own, since the order is the test."""
    import subprocess
    import sys
    code = ("from reef_amd import binding as B\nB.lib()\nimport torch\n"
            "try:\n    B._at(torch.zeros(4))\nexcept RuntimeError as e:\n    assert 'import torch before' in str(e)\nelse:\n    raise SystemExit(3)\n")
    import os
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0, r.stderr


SHARES = r"""
#include <cstdio>
#include "paged_shares.h"
using namespace reef_ops;
// What the wavefronts of the kernel walk over, for one sequence alone: is every token of its window seen, once, and no other?
int main() {
    const int64_t top = 1ll << 31;
    const int64_t lengths[] = {1, 2, 31, 32, 33, 127, 128, 129, 500, 4097, 70001, top - 1, top - 2, top - 31, top - 32, top - 33, top - 128, top - 479, top - 480, top - 512, top - 513};
    const int32_t windows[] = {0, 1, 2, 31, 33, 100, 128, 257, 479, 480, 481, 512, 4000, 100000};
    const int32_t budgets[] = {0, 1, 3, 64, 448, 896};
    for (int64_t length : lengths)
        for (int32_t window : windows)
            for (int32_t budget : budgets)
                for (int waves : {4, 8, 16})
                    for (int tile : {16, 32}) {
                        if (window == 0 && length > 100000 && (budget != 448 || waves != 4 || tile != 32)) continue;    // (many tiles)
                        const int32_t held = (int32_t)length, first = window && held > window ? held - window : 0, n = held - first;
                        const int32_t count = budget ? shares_of(n, tokens_of((float)n, budget)) : 1, stride = waves * tile;
                        if (budget && count > budget + 1) return std::printf("%d shares\n", count), 1;
                        int64_t seen = 0;
                        for (int32_t number = 0; number < count; ++number) {
                            const int32_t begin = first + begin_of(n, number, count), end = number + 1 < count ? first + begin_of(n, number + 1, count) : held;
                            if (begin < first || begin >= end || end > held) return std::printf("share %d of %d: %d %d of %d\n", number, count, begin, end, held), 1;
                            for (int wave = 0; wave < waves; ++wave) {
                                int32_t t0 = first_of(begin, end, wave * tile);
                                while (t0 < end) {
                                    if (t0 < begin || (t0 - begin) % stride != wave * tile) return std::printf("wavefront %d at %d of %d .. %d\n", wave, t0, begin, end), 1;
                                    seen += end - t0 < tile ? end - t0 : tile;
                                    if (t0 >= end - stride) break;
                                    t0 += stride;
                                }
                            }
                        }
                        if (seen != n) return std::printf("%lld of %d seen\n", (long long)seen, n), 1;
                    }
    return 0;
}
"""


def test_shares_cover_sequences_up_to_the_longest(tmp_path):
    """The kernel's own arithmetic, on the host, for lengths just below 2^31 too."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    (tmp_path / "shares.cpp").write_text(SHARES)
    subprocess.check_call(["g++", "-O2", "-fwrapv", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I" + os.path.join(root, "reef_amd", "csrc", "ops"),
                           str(tmp_path / "shares.cpp"), "-o", str(tmp_path / "shares")])
    r = subprocess.run([str(tmp_path / "shares")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout


@pytest.mark.parametrize("scale", [2.4e38, -3.4e38, float("-inf")])
def test_attention_scales_that_are_no_32_bit_number_as_powers_of_two(scale):
    """exp(s) is 2^(s log2 e): the factor of the two has to be finite, or scores of 0 would be NaN."""
    d = attention(layout(), scale=scale)
    refused(call("paged_attention", d, *[P] * 8, 1 << 40), "scale")
    with pytest.raises(B.ReefError):
        B.ops_paged_attention_workspace(d)
    assert B.ops_paged_attention_workspace(attention(layout(), scale=1.7e38)) >= 0


def in_a_process(code):
    import os
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=600, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0, r.stdout + r.stderr


def test_tensors_of_the_host_are_refused():
    """Their addresses would be followed on the device; in a process of its own, which imports torch first."""
    in_a_process("""
import torch
from reef_amd import binding as B
P = 4096
layout = B.CacheLayout(2, 10, 16, 2, 64, 2048, 128, 64)
calls = [(B.ops_block_plan, B.BlockPlanDesc(2, 10, 16, 8, 8, 4, 8), 8),
         (B.ops_cache_append, B.CacheAppendDesc(layout, 2, 3, 128, 64, 128, 64), 5),
         (B.ops_paged_attention, B.PagedAttentionDesc(layout, 2, 2, 8, 4, 4, 0, 0, 0.125, 512, 64, 512, 64), 8),
         (B.ops_beam_select, B.BeamSelectDesc(2, 2, 4, 100, 8, 2, 100), 7),
         (B.ops_beam_reorder, B.BeamReorderDesc(layout, 4, 4, 4, 4, 4, 1, 0), 8)]
for f, desc, n in calls:
    for i in range(n):
        for kind in (torch.int32, torch.bfloat16, torch.float32, torch.uint8):
            args = [P] * n
            if f in (B.ops_paged_attention, B.ops_beam_select):
                args[-1] = None
            args[i] = torch.zeros(64, dtype=kind)
            try:
                f(desc, *args)
            except TypeError as e:
                assert "operand %d: a tensor on the current device" % i in str(e), e
            else:
                raise SystemExit("%s took operand %d of the host" % (f.__name__, i))
try:
    B.ops_cache_append(calls[1][1], P, P, P, P, torch.zeros(64).untyped_storage())
except TypeError as e:
    assert "not on a device" in str(e), e
else:
    raise SystemExit("a storage of the host was taken")
""")


def test_operands_that_are_addresses():
    """Numbers of any kind, c_void_p and None; refused ones come back as the library refuses them."""
    d = append(layout())
    for kind in (int, np.int64, np.uint64, ctypes.c_void_p):
        assert B.ops_cache_append(append(layout(), tokens=0), *[kind(P)] * 5) == 0
        refused(B.ops_cache_append(d, *[kind(P)] * 4, kind(P + 8)), "unaligned")
    refused(B.ops_cache_append(d, P, P, P, P, None), "unaligned")
    for bad in ("x", 1.5, np.zeros(3), [1]):
        with pytest.raises(TypeError):
            B.ops_cache_append(d, P, P, P, P, bad)
    for desc in (None, layout(), B.BlockPlanDesc(2, 10, 16, 8, 8, 4, 8), b"1234"):
        with pytest.raises(TypeError):
            B.ops_cache_append(desc, P, P, P, P, P)


def test_attention_of_more_workgroups_than_a_launch_takes():
    """Refused before the first of its launches."""
    for requests in ((1 << 24) - 1, (1 << 24) - 500):
        d = attention(layout(kv_heads=1), requests=requests, heads=1, max_blocks=1000, table_stride=1000)
        refused(call("paged_attention", d, *[P] * 8, 1 << 60), "too many")


@pytest.mark.parametrize("change", [dict(out_head_stride=0), dict(out_stride=0), dict(out_head_stride=56), dict(out_stride=448), dict(out_stride=64, out_head_stride=64),
                                    dict(out_head_stride=512, out_stride=64, requests=9), dict(heads=2, out_stride=64)])
def test_attention_rows_of_out_that_overlap(change):
    d = attention(layout(), **change)
    refused(call("paged_attention", d, *[P] * 8, 1 << 40), "overlap")
    with pytest.raises(B.ReefError):
        B.ops_paged_attention_workspace(d)


@pytest.mark.parametrize("change", [dict(query_head_stride=0), dict(query_stride=0), dict(out_head_stride=512, out_stride=64, requests=8), dict(requests=1, out_stride=0),
                                    dict(heads=2, out_head_stride=512, out_stride=64), dict(out_stride=2 ** 61), dict(requests=1, heads=2, out_stride=0, out_head_stride=64)])
def test_attention_rows_that_are_apart(change):
    assert B.ops_paged_attention_workspace(attention(layout(), **change)) >= 0
