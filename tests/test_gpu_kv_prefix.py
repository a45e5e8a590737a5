"""kv_prefix_attention against softmax attention over both parts in 64 bits: head
layouts, types, page sizes, lengths of either part from none on, bad pages, unseen
slots, weights, views, other streams, graphs."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from cruise_amd import ops
from kv_ops_reference import wide
from layer_ops_reference import STEP, prefix_attention

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def make(prefix, lengths, heads, kv_heads, d, block, dtype, *, seed=0, spare=2, width=None, prefix_width=None):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    rows = len(lengths)
    width = width if width is not None else max(1, -(-max(lengths, default=0) // block))
    prefix_width = prefix_width if prefix_width is not None else -(-prefix // block)
    pages = prefix_width + rows * width + spare
    order = torch.randperm(pages, generator=gen).int()
    return dict(q=(2 * randn(rows, heads, d)).to(dtype).cuda(), key_cache=randn(pages, block, kv_heads, d).to(dtype).cuda(),
                value_cache=randn(pages, block, kv_heads, d).to(dtype).cuda(), prefix_table=order[:prefix_width].clone().cuda(),
                prefix_length=torch.tensor([prefix], dtype=torch.int32).cuda(),
                block_table=order[prefix_width : prefix_width + rows * width].view(rows, width).clone().cuda(),
                lengths=torch.tensor(lengths, dtype=torch.int32).cuda())


def run(a, weights=True, **more):
    """Calls the operator and compares output and weights; returns the output."""
    pages, block, kv_heads, _ = a["key_cache"].shape
    w = torch.rand(pages, kv_heads, block, device="cuda") if weights else None
    before = wide(w) if weights else None
    out = ops.kv_prefix_attention(**a, weight_cache=w, **more)
    ref, tol, given, given_tol = prefix_attention(a["q"], a["key_cache"], a["value_cache"], a["prefix_table"], a["prefix_length"],
                                                  a["block_table"], a["lengths"], more.get("scale"), more.get("max_prefix"),
                                                  more.get("max_length"))
    off = np.abs(wide(out) - ref)
    assert (off <= tol).all(), (off - tol).max()
    if weights:
        ref = before + given
        assert (np.abs(wide(w) - ref) <= given_tol + STEP * ref).all()
    return out


@pytest.mark.parametrize("heads,kv_heads,d", [(28, 4, 128), (4, 2, 64), (16, 1, 256), (5, 5, 128), (51, 3, 128), (9, 3, 256), (64, 1, 64)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("block", [128, 24, 1])
def test_heads_types_and_pages(heads, kv_heads, d, dtype, block):
    run(make(300, [1, 0, 37, 130], heads, kv_heads, d, block, dtype, seed=heads + block), weights=block != 24)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n", [0, 1, 2, 15, 16, 17, 31, 33, 63, 65, 127, 128, 129, 255, 257, 511, 513, 1023, 1025, 2049, 5000])
def test_prefix_lengths(n, dtype):
    run(make(n, [7, 0, 1], 7, 1, 128, 16, dtype, seed=n))


@pytest.mark.parametrize("block", [16, 24])
@pytest.mark.parametrize("n", [0, 1, 16, 31, 33, 64, 127, 129, 513, 2049, 5000])
@pytest.mark.parametrize("rows,heads,kv_heads,d", [(2, 7, 1, 128), (2, 16, 2, 256), (4, 8, 2, 64), (3, 12, 2, 64)])
def test_prefix_lengths_around_one_tile(rows, heads, kv_heads, d, n, block):
    run(make(n, [7, 0, 130, 1][:rows], heads, kv_heads, d, block, BF16, seed=n), weights=n % 2 == 0)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 9, 10, 17, 18, 19, 33, 64, 65, 74])
def test_rows(rows, dtype):
    """Every number of query tiles, with the last of them full and not."""
    run(make(700, [(5 * r) % 40 for r in range(rows)], 7, 1, 64, 16, dtype, seed=rows))


@pytest.mark.parametrize("heads,kv_heads,d", [(28, 4, 128), (16, 2, 64), (8, 2, 256)])
@pytest.mark.parametrize("block", [128, 100])
def test_many_rows_behind_a_long_prefix(heads, kv_heads, d, block):
    run(make(4000 + block, [60, 0, 11, 33] * 16, heads, kv_heads, d, block, BF16, seed=block))


@pytest.mark.parametrize("block", [3, 16, 100])
def test_long_own_parts(block):
    run(make(1000, [4100, 0, 1, 700, 2048], 14, 2, 64, block, BF16, seed=block))


def test_no_prefix_and_nothing_at_all():
    """Without a prefix it is kv_attention; a row without either gives zeros."""
    a = make(0, [70, 0, 3], 8, 2, 64, 16, BF16, seed=5)
    out = run(a)
    assert bool((out[1] == 0).all())
    alone = {k: v for k, v in a.items() if not k.startswith("prefix")}
    assert torch.allclose(out.float(), ops.kv_attention(**alone).float(), rtol=2**-7, atol=2**-12)
    empty = dict(a, prefix_table=a["prefix_table"][:0], block_table=a["block_table"][:, :0])
    assert bool((ops.kv_prefix_attention(**empty) == 0).all())


@pytest.mark.parametrize("prefix", [2**31 - 1, 70, -5, -(2**31)])
def test_lengths_are_cut(prefix):
    """To what the tables hold and to the bounds, from both ends."""
    a = make(64, [40, 33], 4, 2, 64, 16, F32, seed=6)
    a["prefix_length"][0] = prefix
    a["lengths"][0] = 2**31 - 1
    a["lengths"][1] = -7
    run(a)
    run(a, max_prefix=50, max_length=20)
    run(a, max_prefix=0, max_length=0)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("block", [32, 24])
def test_unseen_slots_may_hold_anything(dtype, block):
    """NaN and infinities behind the lengths and on pages of nobody reach nothing."""
    a = make(300, [20, 0, 5, 64], 8, 2, 128, block, dtype, seed=1, width=9, prefix_width=20)
    want = run(a)
    pages = a["key_cache"].shape[0]
    seen = torch.zeros(pages, block, dtype=torch.bool)
    for table, n in [(a["prefix_table"], 300), *zip(a["block_table"], a["lengths"].tolist())]:
        for j in range(n):
            seen[int(table[j // block]), j % block] = True
    for bad in (float("nan"), float("inf"), float("-inf")):
        for cache in (a["key_cache"], a["value_cache"]):
            cache[~seen.cuda()] = bad
        assert torch.equal(ops.kv_prefix_attention(**a), want)


@pytest.mark.parametrize("block", [16, 24])
def test_bad_pages_are_absent(block):
    a = make(1500, [100, 700, 90, 64], 6, 2, 64, block, BF16, seed=2)
    pages = a["key_cache"].shape[0]
    a["prefix_table"][0], a["prefix_table"][7], a["prefix_table"][20:31] = -1, pages, 2**31 - 1
    a["block_table"][0, 0], a["block_table"][1, 2], a["block_table"][2] = -1, pages, -(2**31)
    run(a)
    a["prefix_table"][:] = -3
    out = run(a)
    assert bool((out[2] == 0).all())


WIDE = [(6, 7, 1, 128, 32), (21, 8, 2, 64, 24), (20, 28, 4, 128, 100), (11, 10, 1, 256, 16), (33, 2, 1, 64, 16), (40, 4, 1, 128, 16)]


@pytest.mark.parametrize("rows,heads,kv_heads,d,block", WIDE)
def test_many_queries_and_unseen_slots(rows, heads, kv_heads, d, block):
    """The same as above where the rows' queries fill whole workgroups."""
    a = make(333, [(7 * r) % 41 for r in range(rows)], heads, kv_heads, d, block, BF16, seed=rows, prefix_width=-(-333 // block) + 3)
    want = run(a)
    pages = a["key_cache"].shape[0]
    seen = torch.zeros(pages, block, dtype=torch.bool)
    for table, n in [(a["prefix_table"], 333), *zip(a["block_table"], a["lengths"].tolist())]:
        for j in range(n):
            seen[int(table[j // block]), j % block] = True
    for bad in (float("nan"), float("inf"), float("-inf")):
        for cache in (a["key_cache"], a["value_cache"]):
            cache[~seen.cuda()] = bad
        assert torch.equal(ops.kv_prefix_attention(**a), want)


@pytest.mark.parametrize("rows,heads,kv_heads,d,block", WIDE)
def test_many_queries_and_bad_pages(rows, heads, kv_heads, d, block):
    a = make(900, [20 + r for r in range(rows)], heads, kv_heads, d, block, BF16, seed=rows + 1)
    pages, width = a["key_cache"].shape[0], a["prefix_table"].shape[0]
    a["prefix_table"][0], a["prefix_table"][width // 2 : width // 2 + 3], a["block_table"][3, 0] = -1, pages, 2**31 - 1
    run(a)
    a["prefix_table"][1:] = -7
    run(a)
    a["block_table"][2] = -1
    out = run(a)
    assert bool((out[2] == 0).all())


@pytest.mark.parametrize("scale", [0.0, 0.3, -0.2, 1.5])
@pytest.mark.parametrize("rows,heads,kv_heads,d,block", WIDE[:4])
def test_many_queries_and_scales(rows, heads, kv_heads, d, block, scale):
    """Scores from all equal to far apart, whichever sign: the base follows the greatest."""
    a = make(1100, [5] * rows, heads, kv_heads, d, block, BF16, seed=rows + 2)
    a["key_cache"] *= torch.linspace(0.1, 3, a["key_cache"].shape[0], device="cuda").to(BF16)[:, None, None, None]
    a["prefix_table"] = a["prefix_table"].sort().values
    run(a, scale=scale)


def test_many_queries_and_one_far_score():
    a = make(900, [50] * 24, 2, 1, 128, 16, BF16, seed=3)
    a["q"] *= 100
    for r in range(0, 24, 5):
        a["key_cache"][int(a["prefix_table"][r + 2]), 3, 0] = a["q"][r, 0] / 10
        a["key_cache"][int(a["block_table"][r + 1, 2]), 1, 0] = a["q"][r + 1, 1] / 10
    run(a)


def test_many_queries_and_infinite_values():
    """An infinite value that a query sees comes out as it is; the others' columns stay numbers."""
    for rows in (3, 30):
        a = make(300, [9] * rows, 4, 1, 64, 16, BF16, seed=4)
        a["value_cache"][int(a["prefix_table"][4]), 2, 0, 7] = float("inf")
        out = ops.kv_prefix_attention(**a)
        assert bool((out[..., 7] == float("inf")).all()) and bool(out[..., :7].isfinite().all()) and bool(out[..., 8:].isfinite().all())


def test_one_far_score_decides():
    """A key along a query, in the prefix or among the own slots, takes the whole softmax: nothing overflows."""
    for dtype in (BF16, F32):
        a = make(900, [50, 50], 2, 1, 64, 16, dtype, seed=3)
        a["q"] *= 100
        a["key_cache"][int(a["prefix_table"][30]), 3, 0] = a["q"][0, 0] / 10
        a["key_cache"][int(a["block_table"][1, 2]), 1, 0] = a["q"][1, 1] / 10
        run(a)


def test_scores_of_minus_infinity():
    """Keys that make every score of the prefix -infinity leave the own slots alone."""
    a = make(256, [30, 0], 2, 1, 64, 16, F32, seed=4)
    a["q"][:] = 1
    a["key_cache"][a["prefix_table"].long(), :, :, 0] = float("-inf")
    out = ops.kv_prefix_attention(**a)
    alone = dict(a, prefix_length=torch.zeros_like(a["prefix_length"]))
    assert torch.allclose(out[0], ops.kv_prefix_attention(**alone)[0], rtol=1e-5, atol=1e-6)
    assert bool(out[1].isnan().all())  # -infinity alone: 0 / 0, as a softmax of them is


def test_shared_pages_and_views():
    """Own pages may be named twice without weights; q, caches and out may be views."""
    a = make(200, [60, 60, 60], 8, 2, 64, 16, BF16, seed=7)
    a["block_table"][1] = a["block_table"][0]
    pages, block, kv_heads, d = a["key_cache"].shape
    both = torch.stack([a["key_cache"], a["value_cache"]], dim=3)
    a["key_cache"], a["value_cache"] = both[:, :, :, 0], both[:, :, :, 1]
    wide_q = torch.zeros(3, 12, d, dtype=BF16, device="cuda")
    wide_q[:, 2:10] = a["q"]
    a["q"] = wide_q[:, 2:10]
    want = run(a, weights=False)
    room = torch.full((8, 3, d), 7, dtype=BF16, device="cuda")
    got = ops.kv_prefix_attention(**a, out=room.transpose(0, 1))
    assert got.data_ptr() == room.data_ptr() and torch.equal(room.transpose(0, 1), want)
    assert torch.equal(ops.kv_prefix_attention(**a, out=a["q"]), want) and torch.equal(a["q"], want)


def test_given_scale_and_equal_calls():
    a = make(2100, [60, 1, 300], 28, 4, 128, 128, BF16, seed=8)
    first = run(a, scale=0.05)
    assert torch.equal(ops.kv_prefix_attention(**a, scale=0.05), first)
    run(a, scale=-0.1)
    run(a, scale=0.0)


@pytest.mark.parametrize("pages_far", [False, True])
def test_offsets_beyond_32_bits(pages_far):
    """A pool of more than 2^31 elements, whose far pages hold the prefix or the rows."""
    block, kv_heads, d = 128, 4, 128
    pages = (1 << 31) // (block * kv_heads * d) + 40
    keys = torch.zeros(pages, block, kv_heads, d, dtype=BF16, device="cuda")
    values = torch.zeros(pages, block, kv_heads, d, dtype=BF16, device="cuda")
    far, near = torch.arange(pages - 12, pages, dtype=torch.int32), torch.arange(12, dtype=torch.int32)
    first, second = (far, near) if pages_far else (near, far)
    gen = torch.Generator().manual_seed(11)
    for cache in (keys, values):
        for where in (far, near):
            cache[where.long().cuda()] = torch.randn(12, block, kv_heads, d, generator=gen).to(BF16).cuda()
    a = dict(q=torch.randn(2, 28, d, generator=gen).to(BF16).cuda(), key_cache=keys, value_cache=values, prefix_table=first.cuda(),
             prefix_length=torch.tensor([1500], dtype=torch.int32).cuda(), block_table=second.view(2, 6).cuda(),
             lengths=torch.tensor([700, 100], dtype=torch.int32).cuda())
    got = ops.kv_prefix_attention(**a)
    small = dict(a, key_cache=torch.cat([keys[:12], keys[-12:]]), value_cache=torch.cat([values[:12], values[-12:]]))
    for name in ("prefix_table", "block_table"):
        small[name] = torch.where(a[name] >= 12, a[name] - (pages - 24), a[name])
    assert torch.equal(got, run(small, weights=False))


def test_graphs_follow_their_tensors():
    """A captured call sees lengths, tables and queries as they are at each replay."""
    a = make(3000, [200, 90, 0, 17], 28, 4, 128, 16, BF16, seed=9)
    weights = torch.zeros(*a["key_cache"].shape[:1], 4, 16, device="cuda")
    ops.kv_prefix_attention(**a, weight_cache=weights)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = ops.kv_prefix_attention(**a, weight_cache=weights)
    for prefix, lengths in [(3000, [200, 90, 0, 17]), (1, [0, 0, 3, 200]), (0, [5, 0, 1, 9]), (2999, [1, 2, 3, 4])]:
        a["prefix_length"].fill_(prefix)
        a["lengths"].copy_(torch.tensor(lengths, dtype=torch.int32))
        a["q"].copy_(torch.randn_like(a["q"].float()))
        weights.zero_()
        graph.replay()
        torch.cuda.synchronize()
        again = torch.zeros_like(weights)
        want = ops.kv_prefix_attention(**a, weight_cache=again)
        assert torch.equal(out, want) and torch.equal(weights, again)


def test_two_streams():
    """Calls at once on two streams keep to themselves."""
    cases = [make(2000 + 500 * i, [100, 3, 40], 14, 2, 128, 128, BF16, seed=30 + i) for i in range(2)]
    want = [ops.kv_prefix_attention(**a) for a in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for i, a in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.kv_prefix_attention(**a))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])
