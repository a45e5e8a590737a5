"""int8_linear of up to 64 tokens whose K is cut into ranges, against its exact sums in
64 bits: channels on both sides of every change of the cut, in a workspace that was
full of other numbers, so that no channel passes that was not written."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from cruise_amd import _lib, ops
from kv_ops_reference import cpu, wide
from layer_ops_reference import product

pytestmark = pytest.mark.gpu
BF16, F32, I8 = torch.bfloat16, torch.float32, torch.int8


def make(tokens, inner, outer, seed, bias):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.rand(*s, generator=gen, device="cuda")  # noqa: E731
    byte = lambda *s: torch.randint(-127, 128, s, generator=gen, device="cuda", dtype=I8)  # noqa: E731
    return dict(x=byte(tokens, inner), x_scale=0.01 * rand(tokens), weight=byte(outer, inner), weight_scale=0.01 * rand(outer),
                bias=rand(outer) if bias else None)


def call(a, fill):
    """The C entry with a workspace and an output that hold `fill` in every byte."""
    tokens, inner = a["x"].shape
    outer = a["weight"].shape[0]
    out = torch.full((tokens, outer * 4), fill, dtype=torch.uint8, device="cuda").view(F32)
    fields = [a["x"].data_ptr(), a["x_scale"].data_ptr(), a["weight"].data_ptr(), a["weight_scale"].data_ptr(),
              0 if a["bias"] is None else a["bias"].data_ptr(), out.data_ptr(), 0, 0, inner, inner, outer, tokens, inner, outer, 1, 4,
              out.get_device()]
    lib = _lib.load()
    need = lib.resident_int8_linear_workspace(ops.INT8_LINEAR.pack(*fields))
    assert need >= 0
    workspace = torch.full((max(need, 16),), fill, dtype=torch.uint8, device="cuda")
    fields[6:8] = workspace.data_ptr(), need
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.resident_int8_linear(ops.INT8_LINEAR.pack(*fields), stream) == 0
    return out, need


def compare(tokens, inner, outer, *, ranges=None, bias=True):
    a = make(tokens, inner, outer, tokens + inner + outer, bias)
    ref, tol = product(cpu(a["x"]).numpy(), cpu(a["x_scale"]).numpy(), a["weight"], a["weight_scale"], a["bias"], F32)
    for fill in (0x5B, 0xA4):  # as whole numbers and as floats both large
        out, need = call(a, fill)
        if ranges is not None:
            assert need == ranges * tokens * ((outer + 3) // 4 * 16)  # the case is the one it is meant to be
        off = np.abs(wide(out) - ref) - tol
        assert (off <= 0).all(), (off.max(), np.unique(np.nonzero(off > 0)[1])[:20])


@pytest.mark.parametrize("tokens,inner,outer,ranges", [
    (48, 28672, 8192, 3), (33, 29568, 8192, 3), (40, 18944, 8192, 3), (64, 14336, 8190, 3), (64, 16384, 8192, 3), (64, 28672, 4096, 6),
    (64, 24576, 4900, 5), (64, 131056, 910, 27), (64, 18944, 3584, 4), (64, 32768, 2048, 6), (49, 18944, 7168, 4)])
def test_long_sums_of_many_channels(tokens, inner, outer, ranges):
    compare(tokens, inner, outer, ranges=ranges)


# 64 tokens of 14,336: three ranges in one round of workgroups up to 8,160 channels, 96 each,
# in two from there; two ranges from 10,753, one from 16,385.
@pytest.mark.parametrize("outer", [95, 96, 97, 255, 256, 257, 1360, 1361, 4080, 4081, 8159, 8160, 8161, 8193, 10752, 10753, 16384, 16385])
def test_channels_around_a_change_of_the_cut(outer):
    compare(64, 14336, outer, bias=outer % 2 == 1)


@pytest.mark.parametrize("tokens", [1, 4, 8, 9, 16, 17, 32, 33, 63, 64])
@pytest.mark.parametrize("inner,outer", [(18944, 3584), (28672, 911), (131056, 257)])
def test_few_tokens_of_long_sums(tokens, inner, outer):
    compare(tokens, inner, outer)
