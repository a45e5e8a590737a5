"""kv_attention against softmax attention in 64 bits: head layouts, types, page
sizes, lengths from none to several thousand, bad pages, what lies in slots that
a row does not see, views, far offsets, graphs."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from cruise_amd import ops
from kv_ops_reference import attention, weights_after, wide

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def make(lengths, heads, kv_heads, d, block, dtype, *, seed=0, spare=2, spread=2.0, width=None):
    gen = torch.Generator().manual_seed(seed)
    width = width or max(1, -(-max(lengths) // block))
    rows = len(lengths)
    pages = rows * width + spare
    randn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return dict(q=(spread * randn(rows, heads, d)).to(dtype).cuda(), key_cache=randn(pages, block, kv_heads, d).to(dtype).cuda(),
                value_cache=randn(pages, block, kv_heads, d).to(dtype).cuda(),
                block_table=torch.randperm(pages, generator=gen)[: rows * width].int().view(rows, width).cuda(),
                lengths=torch.tensor(lengths, dtype=torch.int32).cuda())


def run(a, weights=True, **more):
    """Calls the operator and compares output and weights; returns the output."""
    pages, block, kv_heads, _ = a["key_cache"].shape
    w = torch.rand(pages, kv_heads, block, device="cuda") if weights else None
    before = w.clone() if weights else None
    out = ops.kv_attention(**a, weight_cache=w, **more)
    ref, tol, p = attention(a["q"], a["key_cache"], a["value_cache"], a["block_table"], a["lengths"], more.get("scale"), more.get("max_length"))
    assert (np.abs(wide(out) - ref) <= tol).all(), np.abs(wide(out) - ref).max()
    if weights:
        ref, tol = weights_after(before, p, kv_heads)
        assert (np.abs(wide(w) - ref) <= tol).all(), np.abs(wide(w) - ref).max()
    return out


@pytest.mark.parametrize("heads,kv_heads,d", [(28, 4, 128), (4, 2, 64), (16, 1, 256), (5, 5, 128), (32, 1, 64), (51, 3, 128), (2, 1, 256)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("block", [128, 24, 1])
def test_heads_types_and_pages(heads, kv_heads, d, dtype, block):
    run(make([1, 0, 37, 300, 128], heads, kv_heads, d, block, dtype, seed=heads + block), weights=block != 24)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n", [2, 15, 16, 17, 31, 32, 33, 63, 64, 127, 129, 255, 257, 511, 513, 1023, 1025, 2049, 5000])
def test_lengths(n, dtype):
    run(make([n, n - 1, 1], 7, 1, 128, 16, dtype, seed=n))


@pytest.mark.parametrize("block", [3, 16, 48, 100, 256])
def test_long_rows_beside_short_and_empty_ones(block):
    run(make([4100, 0, 1, 700, 33, 2048], 14, 2, 64, block, BF16, seed=block))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_unseen_slots_may_hold_anything(dtype):
    """NaN and infinities behind the lengths and on pages of no row reach nothing."""
    a = make([200, 5, 0, 64], 8, 2, 128, 32, dtype, seed=1, width=9)
    want = run(a)
    pages, block = a["key_cache"].shape[:2]
    seen = torch.zeros(pages, block, dtype=torch.bool)
    for r, n in enumerate(a["lengths"].tolist()):
        for j in range(n):
            seen[int(a["block_table"][r, j // block]), j % block] = True
    for i, cache in enumerate((a["key_cache"], a["value_cache"])):
        cache[~seen.cuda()] = [float("nan"), float("inf")][i]
    got = ops.kv_attention(**a)
    assert torch.equal(got, want)
    for i, cache in enumerate((a["key_cache"], a["value_cache"])):
        cache[~seen.cuda()] = [float("-inf"), float("nan")][i]
    assert torch.equal(ops.kv_attention(**a), want)


@pytest.mark.parametrize("block", [16, 24])
def test_bad_pages_are_absent(block):
    """Pages outside the pool: first, in the middle, all of a row's."""
    a = make([100, 700, 90, 64], 6, 2, 64, block, BF16, seed=2)
    pages = a["key_cache"].shape[0]
    a["block_table"][0, 0], a["block_table"][1, 2], a["block_table"][1, 5] = -1, pages, 2**31 - 1
    a["block_table"][2] = -(2**31)
    out = run(a)
    assert bool((out[2] == 0).all())


def test_whole_pieces_of_a_row_on_bad_pages():
    """Runs of several hundred absent slots: at the start, in the middle, at the end, and all but one slot."""
    a = make([1500, 1500, 1500, 1500, 2100], 4, 2, 64, 16, BF16, seed=20)
    table = a["block_table"]
    table[0, :40] = -1
    table[1, 16:48] = -1
    table[2, 20:] = -1
    table[3] = torch.where(torch.arange(table.shape[1], device="cuda") == 50, table[3], -1)
    run(a)


@pytest.mark.parametrize("bound", [5000, 20000, 100000])
def test_short_rows_in_a_call_for_long_ones(bound):
    """Rows are cut by what they have, whatever the call is sized for."""
    for lengths in ([900], [3000, 128, 0, 129, 1]):
        run(make(lengths, 4, 2, 64, 16, BF16, seed=22, width=-(-bound // 16), spare=0))


@pytest.mark.parametrize("heads,kv_heads,d,block,n", [(1, 1, 64, 24, 4000), (16, 2, 128, 16, 1000), (7, 1, 128, 5, 1010), (3, 1, 256, 48, 2500)])
def test_whole_rows_of_a_large_batch(heads, kv_heads, d, block, n):
    """As many rows as there are CUs are not cut: a workgroup goes over all of one, its scores in LDS or in memory."""
    a = make([n, n - 1, 17, n // 2], heads, kv_heads, d, block, BF16, seed=n)
    more = 256 // kv_heads
    a["q"] = a["q"].repeat(more // 4, 1, 1)
    for name in ("block_table", "lengths"):
        a[name] = torch.cat([a[name], torch.zeros(more - 4, *a[name].shape[1:], dtype=torch.int32, device="cuda")])
    run(a)


def test_many_short_rows():
    a = make([1 + r % 3 for r in range(3000)], 4, 2, 64, 4, F32, seed=21)
    run(a)


def test_lengths_are_cut():
    a = make([500, 37, 9], 4, 2, 64, 16, BF16, seed=3)
    a["lengths"] = torch.tensor([2**31 - 1, -5, 9], dtype=torch.int32).cuda()
    run(a)
    run(a, max_length=33)
    out = run(a, max_length=0)
    assert bool((out == 0).all())


def test_max_length_does_not_change_results_of_shorter_rows():
    a = make([40, 33, 64], 8, 2, 128, 16, BF16, seed=4, width=300)
    run(a)
    run(a, max_length=64)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_large_scores(dtype):
    """Scores far apart: the maximum decides, nothing overflows."""
    a = make([300, 33], 7, 1, 128, 16, dtype, seed=5, spread=60.0)
    run(a)
    run(make([300, 33], 7, 1, 128, 16, dtype, seed=6), scale=0.0)
    run(make([300, 33], 7, 1, 128, 16, dtype, seed=6), scale=-0.3)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rising_scores(dtype):
    """Every slot's score is above the one before: the running maximum moves at every step."""
    a = make([1500], 4, 2, 64, 16, dtype, seed=7)
    ramp = torch.linspace(-8, 8, 1504, device="cuda").view(-1, 16, 1)
    a["key_cache"].zero_()
    a["key_cache"][a["block_table"][0].long(), :, :, 0] = ramp.expand(-1, 16, 2).to(dtype)
    a["q"].zero_()
    a["q"][:, :, 0] = 16
    run(a)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lengths,block", [([300, 33, 0, 1], 16), ([5000, 700], 24)])
def test_bf16_probabilities_lose_no_bits(d, lengths, block):
    """The stored type rounds the output alone: a probability is off by 2^-15 of
    itself in the product with the values, whatever cancels there."""
    a = make(lengths, 14, 2, d, block, BF16, seed=d)
    ref, tol, _ = attention(a["q"], a["key_cache"], a["value_cache"], a["block_table"], a["lengths"])
    size, _, _ = attention(a["q"], a["key_cache"], a["value_cache"].abs(), a["block_table"], a["lengths"])
    tol = tol - (2.0**-8 - 2.0**-15) * size * (1 + 2.0**-8)  # instead of a rounding of every probability to bf16
    error = np.abs(wide(ops.kv_attention(**a)) - ref)
    assert (error <= tol).all(), (error - tol).max()


@pytest.mark.parametrize("heads,kv_heads,d", [(4, 2, 64), (28, 4, 128), (9, 3, 256)])
def test_fp32_error_on_average(heads, kv_heads, d):
    """Scores of spread 2, of which those that count are seldom above 8: two half
    steps of such a score are 2^-20, and the output's error stays below, taken
    over all of it."""
    a = make([842] * 11, heads, kv_heads, d, 16, F32, seed=26)
    ref, _, _ = attention(a["q"], a["key_cache"], a["value_cache"], a["block_table"], a["lengths"])
    error = wide(ops.kv_attention(**a)) - ref
    assert np.linalg.norm(error) <= 2.0**-20 * np.linalg.norm(ref)


def test_infinite_values_of_small_weight():
    """An infinite value gives infinity, however small its weight or exact in bf16 (2^-k)."""
    a = make([32] * 8, 1, 1, 64, 16, BF16, seed=23)
    a["key_cache"].zero_(), a["q"].zero_()
    a["q"][:, 0, 0] = 1.0
    for r in range(8):
        page = int(a["block_table"][r, 0])
        a["key_cache"][page, 5, 0, 0] = -(0.0, 1.0, 2.0, 8.0, 20.5, 50.0, 70.0, 100.0)[r]
        a["value_cache"][page, 5, 0, r] = float("inf") if r % 2 else float("-inf")
    # the softmax of base 2: weights are 2^-k times those of the others
    out = ops.kv_attention(**a, scale=float(np.log(2.0)))
    want = torch.tensor([float("inf") if r % 2 else float("-inf") for r in range(8)])
    assert torch.equal(out[:, 0].diagonal().float().cpu(), want) and int((~out.isfinite()).sum()) == 8


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_nan_and_infinity_in_seen_slots(dtype):
    """As the formula: a NaN key spoils its row's KV head, an infinite value its
    column; a key of -infinity has no weight, and a row of them no softmax."""
    a = make([70, 70, 70, 40], 4, 2, 64, 16, dtype, seed=8)
    at = lambda r, j: (int(a["block_table"][r, j // 16]), j % 16)  # noqa: E731
    a["key_cache"][at(0, 69)][0, 3] = float("nan")
    a["value_cache"][at(1, 20)][1, 7] = float("inf")
    a["q"][2:] = a["q"][2:].abs()
    for j in range(40):
        a["key_cache"][at(3, j)][0, :] = float("-inf")
        if j < 20:
            a["key_cache"][at(2, j)][0, :] = float("-inf")
    out = ops.kv_attention(**a)
    assert bool(out[0, :2].isnan().all()) and bool(out[0, 2:].isfinite().all())
    assert bool((out[1, 2:, 7] == float("inf")).all()) and int(out[1].isinf().sum()) == 2
    assert bool(out[2].isfinite().all())
    assert bool(out[3, :2].isnan().all()) and bool(out[3, 2:].isfinite().all())
    a["lengths"][2] = 20
    assert bool(ops.kv_attention(**a)[2, :2].isnan().all())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_views(dtype):
    """Caches as a layer of many with heads outside the slots, queries as part of
    a projection's output, a table and weights with wider rows, output in place."""
    a = make([90, 17, 200], 6, 3, 64, 8, dtype, seed=9)
    pages = a["key_cache"].shape[0]
    big = torch.randn(pages, 2, 2, 3, 8, 64, device="cuda").to(dtype)
    a["key_cache"], a["value_cache"] = big[:, 1, 0].transpose(1, 2), big[:, 0, 1].transpose(1, 2)
    qkv = torch.randn(3, 12, 64, device="cuda").to(dtype)
    a["q"] = qkv[:, :6]
    table = torch.full((3, 40), -1, dtype=torch.int32, device="cuda")
    table[:, : a["block_table"].shape[1]] = a["block_table"]
    a["block_table"] = table
    weights = torch.zeros(pages, 2, 3, 8, device="cuda")
    out = ops.kv_attention(**a, weight_cache=weights[:, 1])
    ref, tol, p = attention(a["q"], a["key_cache"], a["value_cache"], a["block_table"], a["lengths"])
    assert (np.abs(wide(out) - ref) <= tol).all()
    ref_w, tol_w = weights_after(torch.zeros(pages, 3, 8), p, 3)
    assert (np.abs(wide(weights[:, 1]) - ref_w) <= tol_w).all() and bool((weights[:, 0] == 0).all())
    same = ops.kv_attention(**a, out=a["q"])
    assert same.data_ptr() == a["q"].data_ptr() and torch.equal(same, out)


def test_pages_beyond_32_bit_offsets():
    """The pool's last pages lie more than 2^31 elements behind its start."""
    block, kv_heads, d = 16, 2, 128
    pages = (1 << 31) // (block * kv_heads * d) + 40
    keys = torch.empty(pages, block, kv_heads, d, dtype=BF16, device="cuda")
    values = torch.empty_like(keys)
    small = make([130, 50], 8, kv_heads, d, block, BF16, seed=10)
    table = small["block_table"].long()
    far = torch.arange(pages - table.numel(), pages, device="cuda").view(table.shape)
    keys[far], values[far] = small["key_cache"][table], small["value_cache"][table]
    want = ops.kv_attention(**small)
    got = ops.kv_attention(small["q"], keys, values, far.int(), small["lengths"])
    assert torch.equal(got, want)


def test_empty_batch_and_table():
    a = make([5], 4, 2, 64, 16, F32)
    assert ops.kv_attention(a["q"][:0], a["key_cache"], a["value_cache"], a["block_table"][:0], a["lengths"][:0]).shape == (0, 4, 64)
    out = ops.kv_attention(a["q"], a["key_cache"], a["value_cache"], a["block_table"][:, :0], a["lengths"])
    assert bool((out == 0).all())


def test_repeats_are_identical():
    a = make([3000, 17, 900], 14, 2, 128, 16, BF16, seed=11)
    results = []
    for _ in range(3):
        w = torch.zeros(a["key_cache"].shape[0], 2, 16, device="cuda")
        results.append((ops.kv_attention(**a, weight_cache=w), w))
    assert all(torch.equal(x, y) for r in results[1:] for x, y in zip(results[0], r))


def test_two_graphs_and_another_stream():
    """Two captured calls with workspaces of their own, replayed in turn and at the same time as eager work."""
    first, second = make([2500, 300], 14, 2, 128, 16, BF16, seed=12), make([1900, 2048, 1], 4, 2, 64, 16, F32, seed=13)
    graphs, outs, weights = [], [], []
    stream = torch.cuda.Stream()
    for a in (first, second):
        w = torch.zeros(a["key_cache"].shape[0], 2, 16, device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = ops.kv_attention(**a, weight_cache=w)
        graphs.append(graph), outs.append(out), weights.append(w)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for step in range(3):
        for a, w in zip((first, second), weights):
            a["q"].normal_()
            a["lengths"].sub_(step)
            a["lengths"].clamp_(min=0)
            w.zero_()
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for a, out, w in zip((first, second), outs, weights):
            eager_w = torch.zeros_like(w)
            assert torch.equal(out, ops.kv_attention(**a, weight_cache=eager_w)) and torch.equal(w, eager_w)
            ref, tol, p = attention(a["q"], a["key_cache"], a["value_cache"], a["block_table"], a["lengths"])
            assert (np.abs(wide(out) - ref) <= tol).all()


def test_python_refusals():
    a = make([5, 6], 4, 2, 64, 16, BF16)
    for name, bad in (("q", a["q"].float()), ("q", a["q"][:, :3]), ("q", a["q"][..., :32]), ("block_table", a["block_table"].long()),
                      ("block_table", a["block_table"][:1]), ("lengths", a["lengths"].long()), ("lengths", a["lengths"].cpu()),
                      ("value_cache", a["value_cache"].float()), ("key_cache", a["key_cache"].flatten(0, 1)),
                      ("q", a["q"].clone().requires_grad_()), ("key_cache", a["key_cache"].clone().requires_grad_())):
        with pytest.raises(ValueError):
            ops.kv_attention(**{**a, name: bad})
    for more in (dict(max_length=-1), dict(max_length=1.5), dict(scale=1e39), dict(out=a["q"].float()), dict(weight_cache=torch.zeros(1, 2, 16, device="cuda"))):
        with pytest.raises(ValueError):
            ops.kv_attention(**a, **more)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_outputs_beside_and_over_the_queries(dtype):
    """An output that shares the queries' storage is the queries, or lies apart from every one of them."""
    a = make([90, 700, 33], 6, 3, 64, 16, dtype, seed=24)
    want = ops.kv_attention(**a)
    wide_rows = torch.zeros(3, 20, 64, dtype=dtype, device="cuda")  # [out | queries | rest] of a row
    pairs = torch.zeros(3, 6, 2, 64, dtype=dtype, device="cuda")  # queries and outputs head by head
    for q, out in ((wide_rows[:, 6:12], wide_rows[:, :6]), (pairs[:, :, 0], pairs[:, :, 1]), (wide_rows[:, 6:12], wide_rows[:, 13:19])):
        q.copy_(a["q"])
        assert torch.equal(ops.kv_attention(**{**a, "q": q}, out=out), want) and torch.equal(q, a["q"])
    q = wide_rows[:, 6:12]
    for out in (wide_rows[:, 5:11], wide_rows[:, 7:13], wide_rows[:, 6:18:2], wide_rows.flatten()[6 * 64 :][: 3 * 6 * 64].view(3, 6, 64),
                a["q"][:1].expand(3, 6, 64)):
        with pytest.raises(ValueError, match="overlap"):
            ops.kv_attention(**{**a, "q": q}, out=out)
