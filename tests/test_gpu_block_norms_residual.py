"""block_norms without a block before it: the residual comes back as it was, so an
output in its place is refused."""
from __future__ import annotations

import pytest
import torch

from cruise_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens", [1, 5])
def test_no_output_in_the_residual_without_x(tokens, dtype):
    residual, norm = torch.randn(tokens, 520, device="cuda").to(dtype), torch.rand(520, device="cuda").to(dtype)
    before = residual.clone()
    with pytest.raises(ValueError, match="resident_block_norms refused its arguments"):
        ops.block_norms(None, residual, pre_norm=norm, out=residual)
    with pytest.raises(ValueError, match="resident_block_norms refused its arguments"):
        ops.block_norms(None, residual, pre_norm=norm, out=residual.view(torch.int8)[:, :520], quantize=True)
    got, out = ops.block_norms(None, residual, pre_norm=norm)
    into = torch.empty_like(out)
    ops.block_norms(None, residual, pre_norm=norm, out=into)
    assert got is residual and torch.equal(residual, before) and torch.equal(into, out)


def test_outputs_in_the_residual_with_x():
    """With x both places are free, as long as they are two."""
    x, residual, norm = (torch.randn(*s, device="cuda").bfloat16() for s in ((3, 520), (3, 520), (520,)))
    want = ops.block_norms(x, residual, pre_norm=norm)
    into = x.clone(), residual.clone()
    got = ops.block_norms(*into, pre_norm=norm, residual_out=into[0], out=into[1])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[1] is into[1]
    with pytest.raises(ValueError):
        ops.block_norms(x, residual, pre_norm=norm, residual_out=residual, out=residual)
