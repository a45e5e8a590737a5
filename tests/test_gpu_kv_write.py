"""kv_write against the definition in 64 bits: head layouts, types, odd sizes,
views, far positions, padded tokens, repeated launches from a captured graph."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from cruise_amd import ops
from kv_ops_reference import rotated, wide, write_tolerance

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def make(tokens, heads, kv_heads, d, block, dtype, *, norm=True, far=1 << 20, pages=None, seed=0):
    gen = torch.Generator().manual_seed(seed)
    pages = pages or -(-tokens // block) + 2
    qkv = torch.randn(tokens, (heads + 2 * kv_heads) * d, generator=gen).to(dtype).cuda()
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([heads * d, kv_heads * d, kv_heads * d], dim=1))
    cache = lambda: torch.randn(pages, block, kv_heads, d, generator=gen).to(dtype).cuda()  # noqa: E731
    scale = lambda: (1 + 0.2 * torch.randn(d, generator=gen)).to(dtype).cuda() if norm else None  # noqa: E731
    return dict(q=q, k=k, v=v, positions=torch.randint(0, far, (tokens,), generator=gen).cuda(),
                slots=torch.randperm(pages * block, generator=gen)[:tokens].int().cuda(), key_cache=cache(), value_cache=cache(),
                inv_freq=(1e6 ** (-torch.arange(0, d, 2).double() / d)).float().cuda(), q_norm=scale(), k_norm=scale())


def check(a, out, before, eps=1e-6, weights=None, positions=None):
    d, dtype = a["q"].shape[2], a["q"].dtype
    for x, norm, got in ((a["q"], a["q_norm"], out), (a["k"], a["k_norm"], None)):
        ref, size = rotated(x, norm, eps, a["positions"], a["inv_freq"])
        tol = write_tolerance(ref, size, dtype, d)
        if got is not None:
            assert (np.abs(wide(got) - ref) <= tol).all()
        else:
            keys, key_tol = wide(before[0]), 0 * wide(before[0])
            values = wide(before[1])
            block = before[0].shape[1]
            for t, slot in enumerate(a["slots"].tolist()):
                if 0 <= slot < before[0].shape[0] * block:
                    keys[slot // block, slot % block], key_tol[slot // block, slot % block] = ref[t], tol[t]
                    values[slot // block, slot % block] = wide(a["v"])[t]
    assert (np.abs(wide(a["key_cache"]) - keys) <= key_tol).all()
    assert (wide(a["value_cache"]) == values).all()


@pytest.mark.parametrize("heads,kv_heads,d", [(28, 4, 128), (4, 2, 64), (16, 1, 256), (5, 5, 64), (9, 3, 128), (1, 1, 256)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens,block,norm", [(1, 128, True), (7, 1, False), (130, 24, True)])
def test_heads_types_and_sizes(heads, kv_heads, d, dtype, tokens, block, norm):
    a = make(tokens, heads, kv_heads, d, block, dtype, norm=norm, seed=heads + tokens)
    before = a["key_cache"].clone(), a["value_cache"].clone()
    check(a, ops.kv_write(**a), before)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("far", [1, 300, 1 << 20, (1 << 31) - 1])
def test_sines_and_cosines_are_rounded_once(far, d):
    """Without a norm, fp32: y = a c - b s with c and s off by half a step each, a
    rounding of one product and one of the result; the angle in 64 bits is off by
    at most 2^-50 of itself (its products here and in the reference)."""
    a = make(333, 2, 1, d, 16, F32, norm=False, far=far, seed=far % 1000 + d)
    a["q"][:, 0, : d // 2] = 0.0  # a half alone: the sines and the cosines themselves
    a["q"][:, 1, d // 2 :] = 0.0
    a["k"][:, 0, : d // 2] = 1.0
    out = ops.kv_write(**a)
    keys = a["key_cache"].flatten(0, 1)[a["slots"].long()]
    angle = a["positions"].cpu().numpy().astype(np.float64)[:, None] * wide(a["inv_freq"])
    c, s = np.abs(np.cos(angle))[:, None], np.abs(np.sin(angle))[:, None]
    for x, got in ((a["q"], out), (a["k"], keys)):
        ref, size = rotated(x, None, 0.0, a["positions"], a["inv_freq"])
        lo, hi = np.split(np.abs(wide(x)), 2, axis=-1)
        terms = np.concatenate([lo * c + hi * s, hi * c + lo * s], -1)
        tol = 2.0**-24 * (2 * terms + np.abs(ref)) * (1 + 2.0**-20) + 2.0**-50 * np.tile(angle[:, None], 2) * size
        error = np.abs(wide(got) - ref)
        assert (error <= tol).all(), (error - tol).max()


def test_many_tokens_pass_the_grid():
    """More (token, head) pairs than one pass of the grid takes."""
    tokens = 20011
    a = make(tokens, 12, 4, 64, 16, BF16, seed=3)
    before = a["key_cache"].clone(), a["value_cache"].clone()
    out = ops.kv_write(**a)
    ref, size = rotated(a["q"], a["q_norm"], 1e-6, a["positions"], a["inv_freq"])
    assert (np.abs(wide(out) - ref) <= write_tolerance(ref, size, BF16, 64)).all()
    ref, size = rotated(a["k"], a["k_norm"], 1e-6, a["positions"], a["inv_freq"])
    slots = a["slots"].long()
    got = a["key_cache"].flatten(0, 1)[slots]
    assert (np.abs(wide(got) - ref) <= write_tolerance(ref, size, BF16, 64)).all()
    expected = before[1].flatten(0, 1)
    expected[slots] = a["v"]
    assert torch.equal(a["value_cache"].flatten(0, 1), expected)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_padded_tokens_weights_and_positions(dtype):
    a = make(11, 8, 2, 128, 16, dtype, seed=5)
    a["slots"][2], a["slots"][7], a["slots"][10] = -1, 3 * 16, -(2**31)  # the pool has three pages
    weights = torch.rand(3, 2, 16, device="cuda")
    positions = torch.full((3, 2, 16), -7, dtype=torch.int32, device="cuda")
    w, p = weights.clone(), positions.clone()
    before = a["key_cache"].clone(), a["value_cache"].clone()
    check(a, ops.kv_write(**a, weight_cache=weights, position_cache=positions), before)
    for t, slot in enumerate(a["slots"].tolist()):
        if 0 <= slot < 48:
            w[slot // 16, :, slot % 16] = 0
            p[slot // 16, :, slot % 16] = int(a["positions"][t])
    assert torch.equal(weights, w) and torch.equal(positions, p)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_views_and_in_place(dtype):
    """Caches as one layer of several with the heads outside the slots, weights
    as a view, queries rotated in place."""
    a = make(9, 6, 3, 64, 8, dtype, seed=6)
    big = torch.randn(3, 2, 2, 3, 8, 64, device="cuda").to(dtype)  # pages, layers, K/V, heads, slots, d
    before = big.clone()
    a["key_cache"], a["value_cache"] = big[:, 1, 0].transpose(1, 2), big[:, 1, 1].transpose(1, 2)
    a["slots"] = torch.randperm(24)[:9].int().cuda()
    weights = torch.ones(3, 2, 3, 8, device="cuda")
    views = before[:, 1, 0].transpose(1, 2), before[:, 1, 1].transpose(1, 2)
    q = a["q"].clone()
    out = ops.kv_write(**a, weight_cache=weights[:, 1], out=a["q"])
    assert out is a["q"]
    a["q"] = q
    check(a, out, views)
    assert torch.equal(big[:, 0], before[:, 0]) and bool((weights[:, 0] == 1).all())
    assert int((weights[:, 1] == 0).sum()) == 9 * 3


def test_zero_heads_keep_finite_and_nan_stays_in_its_head():
    """A head of zeros has no norm to divide by but eps; a NaN reaches its own head only."""
    a = make(2, 4, 2, 128, 16, BF16, seed=7)
    a["q"][0, 1] = 0
    a["q"][1, 2, 5] = float("nan")
    out = ops.kv_write(**a)
    assert bool((out[0, 1] == 0).all())
    assert bool(out[1, 2].isnan().all()) and int(out.isnan().sum()) == 128


def test_positions_beyond_32_bits_of_angle():
    """Positions near 2^31: 64-bit angles keep the full accuracy."""
    a = make(16, 4, 2, 64, 16, F32, norm=False, seed=8)
    a["positions"] = (1 << 31) - 1 - torch.arange(16, device="cuda") * 7919
    before = a["key_cache"].clone(), a["value_cache"].clone()
    check(a, ops.kv_write(**a), before)


def test_pages_beyond_32_bit_offsets():
    """Slots more than 2^31 elements behind the pool's start get what near ones get."""
    a = make(9, 4, 2, 128, 16, BF16, seed=10)
    q = ops.kv_write(**a)
    near = a["slots"].long()
    pages = (1 << 31) // (16 * 2 * 128) + a["key_cache"].shape[0]
    far = near + (pages - a["key_cache"].shape[0]) * 16
    pools = [torch.empty(pages, 16, 2, 128, dtype=BF16, device="cuda") for _ in range(2)]
    got = ops.kv_write(**{**a, "slots": far.int(), "key_cache": pools[0], "value_cache": pools[1]})
    assert torch.equal(got, q)
    for pool, cache in zip(pools, (a["key_cache"], a["value_cache"])):
        assert torch.equal(pool.flatten(0, 1)[far], cache.flatten(0, 1)[near])


def test_no_tokens():
    a = make(1, 4, 2, 64, 16, F32)
    for name in ("q", "k", "v", "positions", "slots"):
        a[name] = a[name][:0]
    before = a["key_cache"].clone()
    assert ops.kv_write(**a).shape == (0, 4, 64)
    assert torch.equal(before, a["key_cache"])


def test_other_stream_and_graph():
    """The current stream is used, and a captured call replays on new inputs."""
    a = make(4, 28, 4, 128, 128, BF16, seed=9)
    stream = torch.cuda.Stream()
    out = torch.empty_like(a["q"], memory_format=torch.contiguous_format)
    with torch.cuda.stream(stream):
        ops.kv_write(**a, out=out)
        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            ops.kv_write(**a, out=out)
    for step in range(4):
        a["q"].normal_()
        a["k"].normal_()
        a["positions"].random_(0, 1000)
        before = a["key_cache"].clone(), a["value_cache"].clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(a, out, before)


def test_python_refusals():
    a = make(3, 4, 2, 64, 16, BF16)
    for name, bad in (("q", a["q"].float()), ("k", a["k"][:, :1]), ("v", a["v"][:2]), ("positions", a["positions"].int()),
                      ("slots", a["slots"].long()), ("inv_freq", a["inv_freq"][:-1]), ("q_norm", a["q_norm"].float()),
                      ("value_cache", a["value_cache"][:1]), ("key_cache", a["key_cache"][..., :32]),
                      ("key_cache", a["key_cache"].half()), ("q", a["q"].cpu()), ("q", a["q"].transpose(1, 2)),
                      ("q", a["q"].clone().requires_grad_()), ("k_norm", a["k_norm"].clone().requires_grad_()),
                      ("value_cache", a["value_cache"].clone().requires_grad_()), ("eps", 1e39)):
        with pytest.raises(ValueError):
            ops.kv_write(**{**a, name: bad})
    shifted = torch.zeros(3 * 4 * 64 + 8, dtype=BF16, device="cuda")[1 : 1 + 3 * 4 * 64].view(3, 4, 64)
    with pytest.raises(ValueError, match="16 bytes"):
        ops.kv_write(**{**a, "q": shifted})


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_outputs_beside_and_over_the_projection(dtype):
    """Rotated queries go to the queries' place, or to one apart from all of q, k and v."""
    a = make(37, 8, 2, 64, 16, dtype, seed=25)
    want = ops.kv_write(**a)
    rows = torch.zeros(37, 20, 64, dtype=dtype, device="cuda")  # [q | k | v | room for the output]
    for name, at, n in (("q", 0, 8), ("k", 8, 2), ("v", 10, 2)):
        rows[:, at : at + n] = a[name]
        a[name] = rows[:, at : at + n]
    for out in (rows[:, 1:9], rows[:, 8:16], rows[:, 4:12], rows[:, 11:19], rows[:, :16:2], rows.flatten()[: 37 * 512].view(37, 8, 64),
                rows[:1, 12:].expand(37, 8, 64)):
        with pytest.raises(ValueError, match="overlap"):
            ops.kv_write(**a, out=out)
    assert torch.equal(ops.kv_write(**a, out=rows[:, 12:]), want)
    assert torch.equal(ops.kv_write(**a, out=a["q"]), want)
