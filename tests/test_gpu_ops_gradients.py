"""The serving operators have no gradient: every tensor that asks for one, input
or output, is refused by name, forward-mode tangents too, and taken where
gradients are off."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from cruise_amd import ops

pytestmark = pytest.mark.gpu


def cuda(*shape, dtype=torch.float32):
    return torch.ones(*shape, dtype=dtype, device="cuda")


def arguments(name):
    table = torch.arange(2, dtype=torch.int32, device="cuda").view(1, 2)
    lengths = torch.full((1,), 20, dtype=torch.int32, device="cuda")
    cache = dict(key_cache=cuda(2, 16, 2, 64), value_cache=cuda(2, 16, 2, 64), weight_cache=cuda(2, 2, 16))
    positions = torch.zeros(2, 2, 16, dtype=torch.int32, device="cuda")
    if name == "kv_write":
        return dict(cache, q=cuda(1, 4, 64), k=cuda(1, 2, 64), v=cuda(1, 2, 64), positions=cuda(1, dtype=torch.int64), slots=lengths,
                    inv_freq=cuda(32), q_norm=cuda(64), k_norm=cuda(64), out=cuda(1, 4, 64))
    if name == "kv_attention":
        return dict(cache, q=cuda(1, 4, 64), block_table=table, lengths=lengths, out=cuda(1, 4, 64))
    if name == "kv_evict":
        return dict(cache, block_table=table, lengths=lengths, next_positions=lengths.long(), position_cache=positions, budget=8, recent=2)
    return dict(logits=cuda(1, 40), history=cuda(1, 20, dtype=torch.int64), history_lengths=lengths, repetition=cuda(1), presence=cuda(1),
                frequency=cuda(1), bias_ids=cuda(1, 3, dtype=torch.int64), bias_values=cuda(1, 3), out=cuda(1, 40))


CASES = [(name, key) for name, keys in {
    "kv_write": ("q", "k", "v", "inv_freq", "q_norm", "k_norm", "key_cache", "value_cache", "weight_cache", "out"),
    "kv_attention": ("q", "key_cache", "value_cache", "weight_cache", "out"),
    "kv_evict": ("key_cache", "value_cache", "weight_cache"),
    "process_logits": ("logits", "repetition", "presence", "frequency", "bias_values", "out"),
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
