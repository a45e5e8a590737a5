"""Without a block before it the norm's residual is returned as it is: a record whose
output takes its place is refused, without a GPU."""
from __future__ import annotations

import pytest

from test_layer_ops_refusals import AT, lib, record  # noqa: F401 (lib is a fixture)

ALONE = dict(x=0, post_norm=0, gate=0, gs1=0, residual_out=0)  # the norm of the residual alone


@pytest.mark.parametrize("changed", [dict(out=2 * AT), dict(out=2 * AT, tokens=1), dict(out=2 * AT, dtype=4, rs=512, os=512),
                                     dict(out=2 * AT + 1024), dict(out=2 * AT, out_scales=8 * AT)])
def test_the_residual_is_kept(lib, changed):  # noqa: F811
    assert lib.resident_block_norms(record("resident_block_norms", **ALONE, **changed), None) == -1
