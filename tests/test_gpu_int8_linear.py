"""quantize_rows bit for bit, and int8_linear against its exact sums in 64 bits:
types, every edge of the tiles, long sums, views, views that start anywhere, graphs."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from cruise_amd import ops
from kv_ops_reference import cpu, wide
from layer_ops_reference import product, quantized

pytestmark = pytest.mark.gpu
BF16, F32, I8 = torch.bfloat16, torch.float32, torch.int8


def same_rows(x, got=None):
    out, scales = got or ops.quantize_rows(x)
    q, s = quantized(x)
    assert np.array_equal(cpu(scales).numpy(), s, equal_nan=True)
    assert np.array_equal(cpu(out).numpy(), q)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("columns", [1, 3, 4, 7, 8, 63, 64, 65, 512, 513, 1104, 3584, 4096, 8200, 18944, 32768, 65536, 65537, 131072, 300001])
def test_quantized_rows(columns, dtype):
    for rows in (1, 5):
        same_rows(torch.randn(rows, columns, generator=torch.Generator().manual_seed(columns)).to(dtype).cuda())


@pytest.mark.parametrize("rows", [0, 2, 1023, 1024, 4100])
def test_quantized_many_rows(rows):
    for columns in (600, 601):
        same_rows((3 * torch.randn(rows, columns)).bfloat16().cuda())


def test_quantized_values_next_to_borders():
    """Halves of a step, ties to even, denormal rows, zeros, infinities and NaN."""
    x = torch.arange(-127, 128, dtype=F32).cuda() / 2
    x = torch.stack([x, x * 2, x * 3e-39, x * 0, x * 1e38, -x, x / 3, x * 1e-45])
    same_rows(x)
    x[0, 5], x[1, 0], x[2, 200] = float("inf"), float("nan"), float("-inf")
    same_rows(x)
    every = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(BF16).view(256, 256).cuda()
    same_rows(every)
    same_rows(every.flip(1).contiguous())
    same_rows(every.t().contiguous())


def test_quantized_views():
    for dtype in (BF16, F32):
        room = torch.randn(7, 700, device="cuda").to(dtype)
        for at in (0, 1, 8):
            x = room[:, at : at + 512]
            into = torch.full((7, 600), 9, dtype=I8, device="cuda")
            scales = torch.empty(7, device="cuda")
            same_rows(x, ops.quantize_rows(x, out=into[:, at : at + 512], scales=scales))
            into[:, at : at + 512] = 9
            assert bool((into == 9).all())
        same_rows(room[:1].expand(4, 700))


def make(tokens, inner, outer, dtype=BF16, *, bias=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    weight = torch.randint(-127, 128, (outer, inner), generator=gen, dtype=torch.int32).to(I8).cuda()
    return dict(x=randn(tokens, inner).to(dtype).cuda(), weight=weight, weight_scale=(0.01 * torch.rand(outer, generator=gen)).cuda(),
                bias=randn(outer).to(dtype).cuda() if bias else None)


def run(a, dtype=None, **more):
    """Calls the operator on x as it is and on x in 8 bits; returns the output."""
    x8, xs = (a["x"], a["x_scale"]) if a["x"].dtype is I8 else ops.quantize_rows(a["x"])
    dtype = dtype or (a["x"].dtype if a["x"].dtype is not I8 else BF16)
    ref, tol = product(cpu(x8).numpy(), cpu(xs).numpy(), a["weight"], a["weight_scale"], a["bias"], dtype)
    out = ops.int8_linear(**a, **more)
    assert out.dtype is dtype and out.shape == ref.shape
    assert (np.abs(wide(out) - ref) <= tol).all(), (np.abs(wide(out) - ref) - tol).max()
    given = ops.int8_linear(x8, a["weight"], a["weight_scale"], x_scale=xs, bias=a["bias"], dtype=dtype)
    assert torch.equal(out, given)
    return out


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5, 8, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300])
def test_tokens(tokens, dtype):
    run(make(tokens, 1104, 200, dtype, seed=tokens))
    run(make(tokens, 256, 33, dtype, seed=tokens, bias=False))


@pytest.mark.parametrize("outer", [1, 2, 3, 7, 8, 15, 16, 17, 63, 64, 65, 127, 129, 255, 256, 257, 511, 513, 1001])
@pytest.mark.parametrize("tokens", [3, 70, 300])
def test_channels(outer, tokens):
    run(make(tokens, 592, outer, seed=outer))


@pytest.mark.parametrize("inner", [16, 32, 48, 64, 80, 112, 128, 144, 240, 256, 272, 496, 512, 528, 1008, 1024, 2032, 4096, 4112, 18944])
@pytest.mark.parametrize("tokens", [1, 20, 64, 150])
def test_inner(inner, tokens):
    run(make(tokens, inner, 100, F32, seed=inner))


@pytest.mark.parametrize("tokens,inner,outer", [(1000, 3584, 520), (2000, 640, 4608), (513, 18944, 260), (4100, 128, 300), (9000, 64, 40)])
def test_large(tokens, inner, outer):
    run(make(tokens, inner, outer, seed=tokens))


@pytest.mark.parametrize("tokens", [2, 64, 300])
def test_sums_of_greatest_magnitude(tokens):
    """The longest sum of the greatest products fits 32 bits, of -128 as well."""
    inner = (1 << 17) - 16
    x = torch.full((tokens, inner), -128, dtype=I8, device="cuda")
    w = torch.full((20, inner), -128, dtype=I8, device="cuda")
    w[::2] = 127
    x[1::2] = 127
    a = dict(x=x, x_scale=torch.rand(tokens, device="cuda"), weight=w, weight_scale=torch.rand(20, device="cuda"), bias=None)
    ref, tol = product(cpu(x).numpy(), cpu(a["x_scale"]).numpy(), w, a["weight_scale"], None, F32)
    assert (np.abs(wide(ops.int8_linear(**a, dtype=F32)) - ref) <= tol).all()


def test_every_element_counts():
    """One nonzero element in x and one in the weights, everywhere once."""
    inner, outer = 400, 48
    for tokens in (4, 40, 200):
        x = torch.zeros(tokens, inner, dtype=I8, device="cuda")
        x[torch.arange(tokens), torch.arange(tokens) * 7 % inner] = 1 + (torch.arange(tokens) % 100).to(I8).cuda()
        w = torch.randint(-128, 128, (outer, inner), dtype=torch.int32).to(I8).cuda()
        one, steps = torch.ones(outer, device="cuda"), torch.ones(tokens, device="cuda")
        got = ops.int8_linear(x, w, one, x_scale=steps, dtype=F32)
        assert torch.equal(got.cpu(), (x.cpu().float() @ w.cpu().float().T))


@pytest.mark.parametrize("tokens", [3, 64, 300])
def test_views(tokens):
    """x that starts anywhere, weights and 8-bit rows of wider tensors, an output beside other things."""
    a = make(tokens, 528, 130, seed=tokens)
    want = run(a)
    room = torch.full((tokens, 560), float("nan"), dtype=BF16, device="cuda")
    room[:, 3:531] = a["x"]
    weights = torch.full((130, 576), 77, dtype=I8, device="cuda")
    weights[:, 16:544] = a["weight"]
    b = dict(a, x=room[:, 3:531], weight=weights[:, 16:544])
    for at in (0, 5):
        into = torch.full((tokens, 150), 3, dtype=BF16, device="cuda")
        got = ops.int8_linear(**b, out=into[:, at : at + 130])
        assert torch.equal(got, want)
        into[:, at : at + 130] = 3
        assert bool((into == 3).all())
    x8, xs = ops.quantize_rows(a["x"])
    eights = torch.full((tokens, 560), 99, dtype=I8, device="cuda")
    eights[:, 16:544] = x8
    assert torch.equal(ops.int8_linear(eights[:, 16:544], b["weight"], a["weight_scale"], x_scale=xs, bias=a["bias"]), want)
    assert torch.equal(ops.int8_linear(x8[:1].expand(tokens, 528), a["weight"], a["weight_scale"], x_scale=xs[:1].expand(tokens).contiguous(),
                                       bias=a["bias"]), want[:1].expand(tokens, 130))


def test_rows_without_numbers():
    """A NaN or an infinity makes its own row NaN, a row of zeros is the bias."""
    a = make(70, 256, 40)
    want = ops.int8_linear(**a)
    a["x"][3, 5], a["x"][9, 0], a["x"][64] = float("nan"), float("-inf"), 0
    got = ops.int8_linear(**a)
    assert bool(got[3].isnan().all()) and bool(got[9].isnan().all()) and torch.equal(got[64], a["bias"])
    others = [r for r in range(70) if r not in (3, 9, 64)]
    assert torch.equal(got[others], want[others])


@pytest.mark.parametrize("tokens", [4, 64, 300])
def test_graphs(tokens):
    a = make(tokens, 3584, 300)
    ops.int8_linear(**a)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = ops.int8_linear(**a)
    for seed in range(4):
        a["x"].copy_(make(tokens, 3584, 1, seed=seed)["x"])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.int8_linear(**a))


@pytest.mark.parametrize("tokens", [5, 64, 200])
@pytest.mark.parametrize("given,result", [(BF16, F32), (F32, BF16), (I8, F32), (I8, BF16)])
def test_results_of_another_type(tokens, given, result):
    a = make(tokens, 208, 77, F32, seed=tokens)
    a["bias"] = a["bias"].to(result)
    x8, xs = ops.quantize_rows(a["x"] if given is I8 else a["x"].to(given))
    a.update(dict(x=x8, x_scale=xs) if given is I8 else dict(x=a["x"].to(given)))
    ref, tol = product(cpu(x8).numpy(), cpu(xs).numpy(), a["weight"], a["weight_scale"], a["bias"], result)
    for out in (ops.int8_linear(**a, dtype=result), ops.int8_linear(**a, out=torch.empty(tokens, 77, dtype=result, device="cuda"))):
        assert out.dtype is result and (np.abs(wide(out) - ref) <= tol).all()


def test_weights_by_quantised_rows():
    """The product of two quantised matrices is off by what the steps round, no more."""
    gen = torch.Generator().manual_seed(9)
    for tokens in (6, 130):
        x, w = torch.randn(tokens, 512, generator=gen).cuda(), torch.randn(300, 512, generator=gen).cuda()
        weight, scale = ops.quantize_rows(w)
        got = wide(ops.int8_linear(x, weight, scale))
        # half a step of each factor, and half of both
        xs, ws = np.abs(wide(x)).max(1) / 254, np.abs(wide(w)).max(1) / 254
        tol = np.abs(wide(x)).sum(1)[:, None] * ws + xs[:, None] * np.abs(wide(w)).sum(1) + 512 * xs[:, None] * ws
        assert (np.abs(got - wide(x) @ wide(w).T) <= tol * (1 + 2.0**-15)).all()


def test_two_streams():
    cases = [make(t, 1104, 500, seed=t) for t in (60, 70)]
    want = [ops.int8_linear(**a) for a in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for i, a in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.int8_linear(**a))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


def test_offsets_beyond_32_bits():
    """More than 2^31 weights, and more than 2^31 outputs."""
    outer, inner = (1 << 31) // 65536 + 5, 65536
    weight = torch.zeros(outer, inner, dtype=I8, device="cuda")
    a = make(3, inner, 5, F32, bias=False)
    weight[-5:] = a["weight"]
    scale = torch.ones(outer, device="cuda")
    scale[-5:] = a["weight_scale"]
    got = ops.int8_linear(a["x"], weight, scale)
    assert torch.equal(got[:, -5:], ops.int8_linear(**a)) and bool((got[:, :-5] == 0).all())
    del weight
    b = make(16385, 16, 131080, bias=False)
    got = ops.int8_linear(**b)
    part = ops.int8_linear(b["x"][-3:].contiguous(), b["weight"][-9:], b["weight_scale"][-9:])
    assert torch.equal(got[-3:, -9:], part)


def own_bytes(x, weight, scales, bias):
    """The call on x itself and on its bytes: the same numbers, also where there are none."""
    x8, steps = ops.quantize_rows(x)
    got = ops.int8_linear(x, weight, scales, bias=bias, dtype=F32)
    want = ops.int8_linear(x8, weight, scales, x_scale=steps, bias=bias, dtype=F32)
    assert torch.equal(got.view(torch.int32), want.view(torch.int32))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("inner", [16, 112, 128, 1008, 1024, 1040, 2064, 3584, 6000, 12032, 12048, 24064, 24080])
@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5, 8, 9, 15, 16, 17])
def test_tokens_as_they_are_and_as_bytes(tokens, inner, dtype):
    gen = torch.Generator().manual_seed(inner + tokens)
    x = (torch.randn(tokens, inner, generator=gen) * torch.logspace(-3, 3, tokens)[:, None]).to(dtype).cuda()
    for outer in (1, 37, 1601):
        weight = torch.randint(-127, 128, (outer, inner), generator=gen).to(torch.int8).cuda()
        own_bytes(x, weight, torch.rand(outer, generator=gen).cuda(), torch.randn(outer, generator=gen).cuda() if outer == 37 else None)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shift,pad", [(0, 0), (0, 16), (0, 3), (1, 16), (8, 8)])
def test_views_and_rows_without_numbers_as_they_are(shift, pad, dtype):
    gen = torch.Generator().manual_seed(shift + pad)
    wide_x = torch.randn(7, 2000 + pad + shift, generator=gen).to(dtype).cuda()
    x = wide_x[:, shift : shift + 2000]
    x[1] = 0
    x[2, 1999] = float("nan")
    x[3, 0] = float("-inf")
    x[4] = torch.finfo(dtype).tiny
    x[5, 1000] = torch.finfo(dtype).max
    weight = torch.randint(-127, 128, (5000, 2000), generator=gen).to(torch.int8).cuda()
    own_bytes(x, weight, torch.rand(5000, generator=gen).cuda(), None)
