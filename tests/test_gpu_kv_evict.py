"""kv_evict against a slot-by-slot selection: which slots stay, where they go,
ties, protected slots, NaN weights, bad pages, untouched rows, repeated rounds."""
from __future__ import annotations

import pytest
import torch

from cruise_amd import ops
from kv_ops_reference import evict

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def make(lengths, kv_heads, d, block, dtype, *, seed=0, spare=2, levels=None, width=None):
    gen = torch.Generator().manual_seed(seed)
    width = width or max(1, -(-max(lengths) // block))
    rows = len(lengths)
    pages = rows * width + spare
    weights = torch.rand(pages, kv_heads, block, generator=gen).pow(-0.5) - 1
    if levels:
        weights = torch.randint(0, levels, weights.shape, generator=gen).float()
    table = torch.randperm(pages, generator=gen)[: rows * width].int().view(rows, width)
    positions = torch.full(weights.shape, -1, dtype=torch.int32)
    for r, n in enumerate(lengths):  # every KV head holds the row's tokens in an order of its own
        for g in range(kv_heads):
            order = torch.randperm(n, generator=gen).int()
            for j in range(n):
                positions[int(table[r, j // block]), g, j % block] = order[j]
    randn = lambda: torch.randn(pages, block, kv_heads, d, generator=gen).to(dtype).cuda()  # noqa: E731
    return dict(key_cache=randn(), value_cache=randn(), block_table=table.cuda(), lengths=torch.tensor(lengths, dtype=torch.int32).cuda(),
                next_positions=torch.tensor(lengths).cuda(), weight_cache=weights.cuda(), position_cache=positions.cuda())


def bits(t):
    t = t.cpu()
    return t.view({2: torch.int16, 4: torch.int32}[t.element_size()]) if t.is_floating_point() else t


def run(a, budget, recent=0, sinks=0, **more):
    ref = evict(a["key_cache"], a["value_cache"], a["weight_cache"], a["position_cache"], a["block_table"], a["lengths"], a["next_positions"],
                budget, recent, sinks, more.get("max_length"))
    new = ops.kv_evict(**a, budget=budget, recent=recent, sinks=sinks, **more)
    got = (a["key_cache"], a["value_cache"], a["weight_cache"], a["position_cache"], new)
    for name, x, y in zip(("keys", "values", "weights", "positions", "lengths"), got, ref):
        assert torch.equal(bits(x), bits(y)), name
    return new


@pytest.mark.parametrize("kv_heads,d", [(4, 128), (2, 64), (1, 256), (5, 64)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("block", [128, 16, 24, 1])
def test_heads_types_and_pages(kv_heads, d, dtype, block):
    run(make([150, 0, 64, 33, 90], kv_heads, d, block, dtype, seed=d + block), budget=40, recent=7, sinks=2)


@pytest.mark.parametrize("n,budget", [(2, 1), (64, 63), (65, 64), (1000, 1), (1023, 1000), (1025, 1024), (2000, 30), (2049, 2047), (3000, 1500),
                                      (4500, 4000), (4096, 3500), (4097, 3585), (1600, 1088), (1601, 1088), (32768, 32000), (32769, 16384)])
def test_sizes(n, budget):
    run(make([n, n // 2, 1], 2, 64, 16, BF16, seed=n), budget=budget, recent=budget // 3, sinks=min(4, budget - budget // 3))


@pytest.mark.parametrize("levels", [1, 2, 7])
def test_ties_go_to_the_lowest_slot(levels):
    run(make([700, 1500], 2, 64, 16, BF16, seed=levels, levels=levels), budget=300, recent=20, sinks=3)
    run(make([700, 1500], 2, 64, 16, BF16, seed=levels, levels=levels), budget=300)


def test_extreme_weights():
    """NaN (of either sign) above all numbers, infinities, both zeros, negative and tiny weights."""
    a = make([900, 300], 2, 64, 16, F32, seed=3)
    w = a["weight_cache"].view(-1)
    values = torch.tensor([float("nan"), -float("nan"), float("inf"), float("-inf"), 0.0, -0.0, -1.0, 1e-45, -1e-45, 3e38], device="cuda")
    w[: w.numel() // 2] = values[torch.randint(0, 10, (w.numel() // 2,), device="cuda")]
    run(a, budget=200, recent=10, sinks=1)


@pytest.mark.parametrize("n,budget", [(300, 200), (1152, 1024), (4096, 1700), (4101, 3900), (9001, 2000), (33000, 32700), (40000, 9000)])
@pytest.mark.parametrize("recent,sinks", [(0, 0), (60, 4)])
def test_more_nan_weights_than_places(n, budget, recent, sinks):
    """NaN weights on both sides of the places left beside finite ones, in rows of each launch's size."""
    places = budget - recent - sinks
    for nans in (places - 1, places, places + 1, n - recent - sinks - 20):
        a = make([n], 1, 64, 16, BF16, seed=n + nans)
        gen = torch.Generator().manual_seed(nans)
        held = a["position_cache"][a["block_table"][0].long(), 0].flatten()[:n].cpu()
        plain = torch.nonzero((held >= sinks) & (held < n - recent))[:, 0]
        slots = plain[torch.randperm(len(plain), generator=gen)[:nans]]
        a["weight_cache"] += 0.7
        a["weight_cache"][a["block_table"][0, slots // 16].long(), 0, slots % 16] = float("nan")
        run(a, budget=budget, recent=recent, sinks=sinks)


def test_protected_slots_alone_and_more_than_expected():
    """recent + sinks = budget; and positions that repeat, so that more slots are protected than the budget holds."""
    run(make([600], 3, 64, 16, BF16, seed=4), budget=64, recent=60, sinks=4)
    a = make([600], 3, 64, 16, BF16, seed=5)
    a["position_cache"].fill_(599)
    run(a, budget=64, recent=1)
    a = make([600], 3, 64, 16, BF16, seed=6)
    a["position_cache"].fill_(-1)  # nothing protected
    run(a, budget=64, recent=60, sinks=4)


@pytest.mark.parametrize("next_position", [-(2**63), -1, 0, 9, 2**31, 2**40, 2**63 - 1])
def test_next_positions_of_any_size(next_position):
    """Behind every slot's position: all of them are recent; far ahead: none."""
    a = make([300], 2, 64, 16, BF16, seed=16)
    a["next_positions"].fill_(next_position)
    run(a, budget=64, recent=10, sinks=2)


def test_rows_with_bad_pages_stay_as_they_are():
    a = make([300, 300, 300, 40], 2, 64, 16, BF16, seed=7, width=20)
    pages = a["key_cache"].shape[0]
    a["block_table"][0, 0], a["block_table"][1, 18] = pages, -1
    a["block_table"][2, 19] = -5  # behind its length: never looked at
    new = run(a, budget=100, recent=10)
    assert new.tolist() == [300, 300, 100, 40]


def test_lengths_are_cut():
    a = make([500, 37, 64], 2, 64, 16, BF16, seed=8)
    a["lengths"] = torch.tensor([2**31 - 1, -5, 64], dtype=torch.int32).cuda()
    run(a, budget=60, max_length=200)


@pytest.mark.parametrize("budget", [200, 1300])
def test_pages_beyond_32_bit_offsets(budget):
    """Pages more than 2^31 elements behind the pool's start, moved by the selecting workgroup and by a launch of its own."""
    a = make([2100, 1500], 2, 128, 16, BF16, seed=15)
    near = a["block_table"].long()
    pages = (1 << 31) // (16 * 2 * 128) + a["key_cache"].shape[0]
    far = near + pages - a["key_cache"].shape[0]
    b = dict(a, block_table=far.int())
    for name in ("key_cache", "value_cache", "weight_cache", "position_cache"):
        b[name] = torch.zeros(pages, *a[name].shape[1:], dtype=a[name].dtype, device="cuda")
        b[name][far] = a[name][near]
    run(a, budget=budget, recent=30)
    ops.kv_evict(**b, budget=budget, recent=30)
    for name in ("key_cache", "value_cache", "weight_cache", "position_cache"):
        assert torch.equal(b[name][far], a[name][near])


def test_nothing_to_evict():
    a = make([30, 10], 2, 64, 16, BF16, seed=9)
    assert run(a, budget=30).tolist() == [30, 10]
    assert run(a, budget=1 << 30).tolist() == [30, 10]
    empty = ops.kv_evict(**{**a, "block_table": a["block_table"][:0], "lengths": a["lengths"][:0], "next_positions": a["next_positions"][:0]},
                         budget=4, recent=0)
    assert empty.shape == (0,)


def test_long_row():
    """More slots than a workgroup holds at once: order and pairing over many tiles."""
    n = 70001
    a = make([70001], 1, 64, 128, BF16, seed=10)
    run(a, budget=20000, recent=512, sinks=4)
    b = make([n], 1, 64, 100, BF16, seed=11, levels=50)
    run(b, budget=69000)


def test_steady_state_rounds():
    """Rounds of appended tokens and evictions: each works on what the one before left."""
    a = make([100, 80], 2, 64, 16, BF16, seed=12, width=8)
    a["next_positions"] = a["lengths"].long()
    for step in range(6):
        a["lengths"] = run(a, budget=64, recent=16, sinks=2)
        for _ in range(step + 1):
            for r in range(2):
                j = int(a["lengths"][r])
                page, at = int(a["block_table"][r, j // 16]), j % 16
                a["key_cache"][page, at].normal_()
                a["weight_cache"][page, :, at].uniform_()
                a["position_cache"][page, :, at] = int(a["next_positions"][r])
            a["lengths"] += 1
            a["next_positions"] += 1


def test_views():
    a = make([90, 70], 3, 64, 8, F32, seed=13)
    pages = a["key_cache"].shape[0]
    big = torch.randn(pages, 2, 3, 8, 64, device="cuda")
    other = big[:, 0].clone()
    a["key_cache"] = big[:, 1].transpose(1, 2)
    w, p = torch.rand(pages, 2, 3, 8, device="cuda"), torch.zeros(pages, 5, 8, dtype=torch.int32, device="cuda")
    p[:, 1:4] = a["position_cache"]
    a["weight_cache"], a["position_cache"] = w[:, 1], p[:, 1:4]
    run(a, budget=50, recent=9)
    assert torch.equal(big[:, 0], other) and bool((p[:, 0] == 0).all()) and bool((p[:, 4] == 0).all())


def test_graph_replays_on_new_lengths():
    a = make([400, 300], 2, 64, 16, BF16, seed=14)
    fresh = {k: v.clone() for k, v in a.items()}
    out = torch.empty(2, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.kv_evict(**a, budget=100, recent=20, sinks=1, out_lengths=out)
    for lengths in ([400, 300], [100, 101], [399, 0]):
        for k, v in fresh.items():
            a[k].copy_(v)
        a["lengths"].copy_(torch.tensor(lengths))
        a["weight_cache"].uniform_()
        ref = evict(a["key_cache"], a["value_cache"], a["weight_cache"], a["position_cache"], a["block_table"], a["lengths"],
                    a["next_positions"], 100, 20, 1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip((a["key_cache"], a["value_cache"], a["weight_cache"], a["position_cache"], out), ref):
            assert torch.equal(bits(x), bits(y))


def test_python_refusals():
    a = make([50], 2, 64, 16, BF16)
    for bad in (dict(budget=0, recent=0), dict(budget=4, recent=5), dict(budget=4, recent=2, sinks=3), dict(budget=4, recent=-1),
                dict(budget=4, recent=0, max_length=-1), dict(budget=4, recent=0, out_lengths=a["lengths"]), dict(budget=4.5, recent=0),
                dict(budget=4, recent=0.5)):
        with pytest.raises(ValueError):
            ops.kv_evict(**a, **bad)
    for name, bad in (("weight_cache", None), ("position_cache", None), ("weight_cache", a["weight_cache"].double()),
                      ("position_cache", a["position_cache"][:, :1]), ("next_positions", a["lengths"]), ("lengths", a["lengths"].long()),
                      ("block_table", a["block_table"][0])):
        with pytest.raises(ValueError):
            ops.kv_evict(**{**a, name: bad}, budget=4, recent=0)
