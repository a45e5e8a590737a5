"""block_norms against its formula in 64 bits: types, every kind of gate, sizes from
one channel to the largest, rows that start anywhere, in place, to 8 bits, graphs."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from cruise_amd import ops
from kv_ops_reference import HALF_STEP, wide
from layer_ops_reference import STEP, norms

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
GATES = ("none", "channel", "token", "element")


def make(tokens, hidden, dtype, *, post=True, gate="channel", seed=0):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    shape = {"none": None, "channel": (hidden,), "token": (tokens, 1), "element": (tokens, hidden)}[gate]
    return dict(x=randn(tokens, hidden).to(dtype).cuda(), residual=(4 * randn(tokens, hidden)).to(dtype).cuda(),
                pre_norm=(1 + 0.2 * randn(hidden)).to(dtype).cuda(), post_norm=(1 + 0.2 * randn(hidden)).to(dtype).cuda() if post else None,
                gate=None if shape is None else randn(*shape).to(dtype).cuda())


def compare(a, got, quantize=False, **more):
    ref, tol, out, loose = norms(a["x"], a["residual"], a["pre_norm"], a["post_norm"], a["gate"], **more)
    assert (np.abs(wide(got[0]) - ref) <= tol).all(), (np.abs(wide(got[0]) - ref) - tol).max()
    if not quantize:
        half = HALF_STEP[a["residual"].dtype]
        assert (np.abs(wide(got[1]) - out) <= half * np.abs(out) + loose).all()
        return
    step = wide(got[2])[:, None]
    # The scale is the greatest value's, a 127th of it rounded; a value is at most half a step off, and the fp32 quotient that
    # is rounded by 127 of its own half steps.
    assert (np.abs(127 * step - np.abs(out).max(1, keepdims=True)) <= loose.max(1, keepdims=True) + 254 * STEP * step).all()
    assert (np.abs(wide(got[1]) * step - out) <= loose + step * (0.5 + 254 * STEP)).all()


def run(a, quantize=False, **more):
    before = {k: None if v is None else v.clone() for k, v in a.items()}
    got = ops.block_norms(**a, quantize=quantize, **more)
    compare(before, got, quantize, **more)
    assert all(v is None or torch.equal(v, a[k]) for k, v in before.items())
    return got


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("quantize", [False, True])
def test_types_and_gates(dtype, post, gate, quantize):
    for hidden in (3584, 1001):
        run(make(5, hidden, dtype, post=post, gate=gate, seed=hidden), quantize, scale=0.5, eps=1e-5)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hidden", [1, 2, 3, 7, 8, 9, 63, 64, 65, 255, 256, 511, 512, 513, 1024, 2047, 2048, 2056, 4096, 4104, 8191, 8192, 8200,
                                    16383, 16384, 18944, 32767, 32768])
def test_sizes(hidden, dtype):
    for tokens in (1, 3):
        run(make(tokens, hidden, dtype, seed=hidden))
        run(make(tokens, hidden, dtype, seed=hidden, gate="element"), quantize=True)


@pytest.mark.parametrize("tokens", [0, 1, 2, 4, 255, 257, 1023, 1025, 4099])
@pytest.mark.parametrize("hidden", [512, 600, 1001])
def test_many_tokens(tokens, hidden):
    got = run(make(tokens, hidden, BF16, gate="token", seed=tokens))
    assert got[0].shape == got[1].shape == (tokens, hidden)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_no_block(dtype):
    """Without x only the norm: the residual comes back itself."""
    a = dict(make(6, 640, dtype, post=False, gate="none"), x=None)
    got = ops.block_norms(**a)
    assert got[0] is a["residual"]
    compare(a, got)
    compare(a, ops.block_norms(**a, quantize=True), quantize=True)


@pytest.mark.parametrize("hidden", [512, 500, 8192])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_in_place(hidden, dtype):
    """The outputs may take the places of x, the residual or an element gate."""
    for tokens in (2, 1500):
        a = make(tokens, hidden, dtype, gate="element", seed=hidden)
        want = ops.block_norms(**a)
        for residual_out, out in [("residual", "x"), ("x", "residual"), ("gate", "residual"), ("residual", "gate")]:
            b = {k: v.clone() for k, v in a.items()}
            got = ops.block_norms(**b, residual_out=b[residual_out], out=b[out])
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("shift", [0, 1, 3, 8])
def test_views(shift):
    """Rows of wider tensors that start anywhere, broadcast ones, and what lies beside them."""
    tokens, hidden = 9, 520
    for dtype in (BF16, F32):
        a = make(tokens, hidden, dtype, gate="element", seed=shift)

        def inside(t, fill=float("nan")):
            room = torch.full((tokens, hidden + 16 + shift), fill, dtype=t.dtype, device="cuda")
            room[:, shift : shift + hidden] = t
            return room, room[:, shift : shift + hidden]

        b = {k: inside(v)[1] if v.dim() == 2 else v for k, v in a.items()}
        rooms = [inside(torch.zeros(tokens, hidden, dtype=dtype, device="cuda"), 5.0) for _ in range(2)]
        ops.block_norms(**b, residual_out=rooms[0][1], out=rooms[1][1])
        compare(a, [view for _, view in rooms])
        for room, _ in rooms:
            room[:, shift : shift + hidden] = 5
            assert bool((room == 5).all())
        eight = inside(torch.zeros(tokens, hidden, dtype=torch.int8, device="cuda"), 5)
        got = ops.block_norms(**b, quantize=True, out=eight[1])
        compare(a, got, quantize=True)
        eight[1][:] = 5
        assert bool((eight[0] == 5).all())
    one = torch.randn(1, hidden, device="cuda")
    a = dict(make(tokens, hidden, F32, gate="none"), x=one.expand(tokens, hidden))
    compare(a, ops.block_norms(**a))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_of_zeros_and_of_no_numbers(dtype):
    """A row of zeros gives zeros; a NaN or an infinity stays in its row."""
    a = make(5, 256, dtype, gate="none")
    want = ops.block_norms(**a, quantize=True)
    a["x"][1], a["residual"][1] = 0, 0
    a["x"][2, 7], a["residual"][3, 9] = float("nan"), float("inf")
    residual, out = ops.block_norms(**a)
    assert bool((residual[1] == 0).all()) and bool((out[1] == 0).all())
    assert bool(residual[2].isnan().all()) and bool(out[2].isnan().all()) and bool(out[3, 9].isnan())
    residual, eight, scales = ops.block_norms(**a, quantize=True)
    assert scales[1] == 0 and bool(scales[2].isnan()) and bool(scales[3].isnan()) and bool((eight[1:4] == 0).all())
    for r in (0, 4):
        assert torch.equal(eight[r], want[1][r]) and scales[r] == want[2][r]


@pytest.mark.parametrize("quantize", [False, True])
def test_graphs(quantize):
    a = make(33, 3584, BF16, gate="element")
    ops.block_norms(**a, quantize=quantize)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = ops.block_norms(**a, quantize=quantize)
    for seed in range(3):
        a["x"].copy_(make(33, 3584, BF16, gate="element", seed=seed)["x"])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, ops.block_norms(**a, quantize=quantize)))


def test_offsets_beyond_32_bits():
    tokens, hidden = (1 << 31) // 8192 + 3, 8192
    x = torch.zeros(tokens, hidden, dtype=BF16, device="cuda")
    a = make(3, hidden, BF16)
    x[-3:] = a["x"]
    got = ops.block_norms(x, x, pre_norm=a["pre_norm"], quantize=True, residual_out=x)
    compare(dict(a, residual=a["x"], post_norm=None, gate=None), [g[-3:] for g in got], quantize=True)
    assert bool((got[2][:-3] == 0).all())
