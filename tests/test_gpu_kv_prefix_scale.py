"""kv_prefix_attention with a scale of 0: every slot that is there weighs the same,
whatever the keys hold."""
from __future__ import annotations

import pytest
import torch

from test_gpu_kv_prefix import BF16, F32, WIDE, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,heads,kv_heads,d,block", [(2, 7, 1, 128, 16), *WIDE[:4]])
def test_keys_of_any_size(rows, heads, kv_heads, d, block, dtype):
    """Products of up to 10^37, still finite in 32 bits, times 0 are 0."""
    a = make(700, [(3 * r) % 20 for r in range(rows)], heads, kv_heads, d, block, dtype, seed=rows)
    a["key_cache"] *= 2.0**117
    assert bool(a["key_cache"].isfinite().all())
    a["prefix_table"][2] = -1
    run(a, scale=0.0)
    run(a, scale=-0.0)
