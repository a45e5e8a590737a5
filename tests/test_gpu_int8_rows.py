"""int8_linear on bf16 and fp32 rows against a reference that quantises them itself and
sums in 64 bits, and products of more tokens whose K is cut into ranges, in a workspace
that was full of other numbers."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from cruise_amd import ops
from kv_ops_reference import wide
from layer_ops_reference import product, quantized
from test_gpu_int8_ranges import compare

pytestmark = pytest.mark.gpu
BF16, F32, I8 = torch.bfloat16, torch.float32, torch.int8


def against_the_rows(x, weight, scales, bias, result):
    """Rows that hold no number come out as none; the others within the reference's tolerance."""
    x8, steps = quantized(x)
    none = np.isnan(steps)
    ref, tol = product(x8, np.where(none, 0, steps), weight, scales, bias, result)
    got = wide(ops.int8_linear(x, weight, scales, bias=bias, dtype=result))
    assert np.isnan(got[none]).all()
    assert (np.abs(got - ref)[~none] <= tol[~none]).all(), (np.abs(got - ref) - tol)[~none].max()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("inner", [16, 112, 1040, 3584, 12048, 24080])
@pytest.mark.parametrize("tokens", [1, 5, 9, 17, 64])
def test_rows_as_they_are(tokens, inner, dtype):
    gen = torch.Generator().manual_seed(inner + tokens)
    x = (torch.randn(tokens, inner, generator=gen) * torch.logspace(-3, 3, tokens)[:, None]).to(dtype).cuda()
    for outer in (37, 1601):
        weight = torch.randint(-127, 128, (outer, inner), generator=gen).to(I8).cuda()
        bias = torch.randn(outer, generator=gen).to(dtype).cuda() if outer == 37 else None
        against_the_rows(x, weight, torch.rand(outer, generator=gen).cuda(), bias, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens", [7, 90])
@pytest.mark.parametrize("shift,pad", [(0, 16), (0, 3), (1, 16), (8, 8)])
def test_views_and_rows_without_numbers(shift, pad, tokens, dtype):
    gen = torch.Generator().manual_seed(shift + pad)
    x = torch.randn(tokens, 2000 + pad + shift, generator=gen).to(dtype).cuda()[:, shift : shift + 2000]
    x[1] = 0
    x[2, 1999] = float("nan")
    x[3, 0] = float("-inf")
    x[4, :1999] = 0  # one value alone, the greatest of its row
    x[5, 1000] = 1e30
    weight = torch.randint(-127, 128, (500, 2000), generator=gen).to(I8).cuda()
    against_the_rows(x, weight, torch.rand(500, generator=gen).cuda(), None, F32)


@pytest.mark.parametrize("tokens,inner,outer,ranges", [(65, 18944, 260, 50), (150, 18944, 1001, 19), (300, 8192, 513, 13), (129, 131056, 77, 128)])
def test_more_tokens_of_long_sums(tokens, inner, outer, ranges):
    compare(tokens, inner, outer, ranges=ranges)


def test_an_output_that_is_no_tensor_is_refused():
    x, weight = torch.randn(3, 64, device="cuda"), torch.ones(5, 64, dtype=I8, device="cuda")
    for out in (0, [1.0], np.zeros((3, 5))):
        with pytest.raises(ValueError, match="out must be a torch.float32 tensor"):
            ops.int8_linear(x, weight, torch.ones(5, device="cuda"), out=out)
