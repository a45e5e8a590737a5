"""kv_prefix_attention, block_norms, quantize_rows and int8_linear have no gradient:
every tensor that asks for one, input or output, is refused by name, forward-mode
tangents too, and taken where gradients are off.  Shapes and types that do not fit are
refused before anything is queued."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from cruise_amd import ops

pytestmark = pytest.mark.gpu


def cuda(*shape, dtype=torch.float32):
    return torch.ones(*shape, dtype=dtype, device="cuda")


def arguments(name):
    if name == "kv_prefix_attention":
        table = torch.arange(2, dtype=torch.int32, device="cuda")
        return dict(key_cache=cuda(2, 16, 2, 64), value_cache=cuda(2, 16, 2, 64), weight_cache=cuda(2, 2, 16), q=cuda(1, 4, 64),
                    prefix_table=table[:1], prefix_length=cuda(1, dtype=torch.int32), block_table=table[1:].view(1, 1),
                    lengths=cuda(1, dtype=torch.int32), out=cuda(1, 4, 64))
    if name == "block_norms":
        return dict(x=cuda(2, 32), residual=cuda(2, 32), pre_norm=cuda(32), post_norm=cuda(32), gate=cuda(32), residual_out=cuda(2, 32),
                    out=cuda(2, 32))
    if name == "quantize_rows":
        return dict(x=cuda(2, 32), scales=cuda(2))
    return dict(x=cuda(2, 32), weight=cuda(3, 32, dtype=torch.int8), weight_scale=cuda(3), bias=cuda(3), out=cuda(2, 3))


CASES = [(name, key) for name, keys in {
    "kv_prefix_attention": ("q", "key_cache", "value_cache", "weight_cache", "out"),
    "block_norms": ("x", "residual", "pre_norm", "post_norm", "gate", "residual_out", "out"),
    "quantize_rows": ("x", "scales"),
    "int8_linear": ("x", "weight_scale", "bias", "out"),
}.items() for key in keys]


@pytest.mark.parametrize("name,key", CASES)
def test_tensors_that_ask_for_a_gradient(name, key):
    a = arguments(name)
    a[key].requires_grad_()
    with pytest.raises(ValueError, match=f"{key} asks for a gradient"):
        getattr(ops, name)(**a)
    with torch.no_grad():
        getattr(ops, name)(**a)
    torch.cuda.synchronize()


@pytest.mark.parametrize("name,key", CASES)
def test_forward_mode_tangents(name, key):
    a = arguments(name)
    with forward_ad.dual_level():
        getattr(ops, name)(**a)  # a level without tangents changes nothing
        a[key] = forward_ad.make_dual(a[key], torch.ones_like(a[key]))
        with pytest.raises(ValueError, match=f"{key} asks for a gradient"):
            getattr(ops, name)(**a)
    torch.cuda.synchronize()


@pytest.mark.parametrize("name,changed,why", [
    ("kv_prefix_attention", dict(prefix_table=lambda: cuda(3)), "prefix_table"), ("kv_prefix_attention", dict(prefix_length=lambda: cuda(2, dtype=torch.int32)), "prefix_length"),
    ("kv_prefix_attention", dict(max_prefix=lambda: -1), "max_prefix is negative"), ("kv_prefix_attention", dict(q=lambda: cuda(1, 3, 64)), "multiple"),
    ("kv_prefix_attention", dict(max_prefix=lambda: 1.5), "resident_kv_prefix_attention"),
    ("block_norms", dict(x=lambda: cuda(2, 31)), "x has shape"), ("block_norms", dict(gate=lambda: cuda(3, 1)), "gate has shape"),
    ("block_norms", dict(gate=lambda: 2.0), "gate"), ("block_norms", dict(pre_norm=lambda: None), "pre_norm"),
    ("block_norms", dict(out_scales=lambda: cuda(2)), "needs quantize"), ("block_norms", dict(x=lambda: None), "need x"),
    ("block_norms", dict(residual=lambda: cuda(2, 32, dtype=torch.float16)), "residual must be"), ("block_norms", dict(scale=lambda: "1"), "resident_block_norms"),
    ("quantize_rows", dict(x=lambda: cuda(2, 32, dtype=torch.int8)), "x must be"), ("quantize_rows", dict(out=lambda: cuda(2, 32)), "out must be"),
    ("int8_linear", dict(weight=lambda: cuda(3, 33, dtype=torch.int8)), "weight has shape"), ("int8_linear", dict(weight=lambda: cuda(3, 32)), "weight must be"),
    ("int8_linear", dict(x_scale=lambda: cuda(2)), "x_scale belongs"), ("int8_linear", dict(x=lambda: cuda(2, 32, dtype=torch.int8)), "x_scale belongs"),
    ("int8_linear", dict(dtype=lambda: torch.float16, out=lambda: None), "bfloat16 or float32"), ("int8_linear", dict(bias=lambda: cuda(4)), "bias has shape"),
    ("int8_linear", dict(x=lambda: cuda(2, 24), weight=lambda: cuda(3, 24, dtype=torch.int8)), "refused its arguments"),
])
def test_refused(name, changed, why):
    a = {**arguments(name), **{k: make() for k, make in changed.items()}}
    with pytest.raises(ValueError, match=why):
        getattr(ops, name)(**a)


def test_overlaps_are_refused():
    """An output lies over no part of an input that it does not take the place of."""
    room = cuda(4, 64)
    with pytest.raises(ValueError, match="refused"):
        ops.block_norms(room[:2, :32], room[2:, :32], pre_norm=cuda(32), out=room[:2, 16:48])
    with pytest.raises(ValueError, match="refused"):
        ops.block_norms(room[:2, :32], room[2:, :32], pre_norm=cuda(32), residual_out=room[:2, :32], out=room[:2, :32])
    with pytest.raises(ValueError, match="refused"):
        ops.int8_linear(room[:, :32], cuda(32, 32, dtype=torch.int8), cuda(32), out=room[:, 16:48])
    # the other halves of the same rows are apart
    ops.int8_linear(room[:, :32], cuda(32, 32, dtype=torch.int8), cuda(32), out=room[:, 32:])
    ops.block_norms(room[:2, :32], room[2:, :32], pre_norm=cuda(32), out=room[:2, 32:])
    torch.cuda.synchronize()
