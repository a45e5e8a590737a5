"""Records and refusals of kv_prefix_attention, block_norms, quantize_rows and
int8_linear, without a GPU: the packed records have the sizes and field orders of
include/resident_epoch.h, one field of a good record is made bad at a time, and
outputs that overlap what they are made of are refused unless they take its place.
The addresses are never followed on the host, and nothing is launched."""
from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from cruise_amd import _lib, build, ops

HEADER = Path(__file__).resolve().parents[1] / "include" / "resident_epoch.h"
AT = 1 << 20  # an aligned address that nothing follows
FAR = 1 << 30


@pytest.fixture(scope="module")
def lib():
    if not _lib.library_path().is_file():
        build.build()
    return _lib.load()


CACHE = dict(keys=AT, values=AT, weights=AT, positions=0, ks0=16 * 4 * 64, ks1=4 * 64, ks2=64, vs0=16 * 4 * 64, vs1=4 * 64, vs2=64,
             ws0=64, ws1=16, ps0=0, ps1=0, pages=8, block=16, kv_heads=4, head_dim=64, dtype=2, device=-1)
PREFIX = dict(CACHE, q=AT, out=FAR, table=AT, lengths=AT, workspace=AT, workspace_bytes=1 << 30, qs0=512, qs1=64, os0=512, os1=64,
              table_stride=4, rows=2, heads=8, width=4, max_length=64, scale=0.125, reserved=0, prefix_table=AT, prefix_length=AT,
              prefix_width=4, max_prefix=64)
NORMS = dict(x=AT, residual=2 * AT, post_norm=3 * AT, gate=4 * AT, pre_norm=5 * AT, residual_out=6 * AT, out=7 * AT, out_scales=0, xs=512, rs=512,
             ros=512, os=512, gs0=0, gs1=1, tokens=5, hidden=512, dtype=2, device=-1, eps=1e-6, scale=1.0)
ROWS = dict(x=AT, out=2 * AT, scales=3 * AT, xs=512, os=512, rows=5, columns=512, dtype=2, device=-1)
LINEAR = dict(x=AT, x_scales=0, weight=2 * AT, weight_scales=3 * AT, bias=4 * AT, out=5 * AT, workspace=FAR, workspace_bytes=1 << 20, xs=512,
              ws=512, os=256, tokens=5, inner=512, outer=256, x_bytes=2, out_bytes=2, device=-1)
ENTRIES = {
    "resident_kv_prefix_attention": (ops.KV_PREFIX_ATTENTION, PREFIX, "ResidentKvPrefixAttention"),
    "resident_block_norms": (ops.BLOCK_NORMS, NORMS, "ResidentBlockNorms"),
    "resident_quantize_rows": (ops.QUANTIZE_ROWS, ROWS, "ResidentQuantizeRows"),
    "resident_int8_linear": (ops.INT8_LINEAR, LINEAR, "ResidentInt8Linear"),
}
BAD = {
    "resident_kv_prefix_attention": [
        ("keys", 0), ("values", AT + 2), ("ks1", -64), ("vs2", 4), ("pages", 0), ("block", 0), ("head_dim", 96), ("dtype", 1), ("q", 0),
        ("out", 0), ("table", 0), ("lengths", 0), ("q", AT + 8), ("out", AT + 64), ("qs0", 4), ("os1", 12), ("table_stride", -1), ("rows", -1),
        ("heads", 6), ("width", -1), ("max_length", -1), ("workspace", 0), ("workspace", AT + 4), ("workspace_bytes", -1), ("workspace_bytes", 64),
        ("reserved", 1), ("prefix_table", 0), ("prefix_length", 0), ("prefix_table", AT + 2), ("prefix_length", AT + 1), ("prefix_width", -1),
        ("max_prefix", -1)],
    "resident_block_norms": [
        ("x", AT + 1), ("residual", 0), ("residual", 2 * AT + 1), ("pre_norm", 0), ("pre_norm", 5 * AT + 1), ("post_norm", 3 * AT + 1),
        ("gate", 4 * AT + 1), ("residual_out", 0), ("out", 0), ("out", 7 * AT + 1), ("x", 0), ("out_scales", 8 * AT + 2), ("xs", -1), ("rs", -1),
        ("ros", -512), ("os", 511), ("gs0", -1), ("gs1", 2), ("gs1", -1), ("tokens", -1), ("hidden", 0), ("hidden", 32769), ("dtype", 1),
        ("eps", -1.0), ("eps", float("nan")), ("scale", float("nan")),
        # outputs over inputs that they do not take the place of, over each other, over the weights
        ("out", AT + 512), ("out", 6 * AT), ("out", 6 * AT + 16), ("residual_out", 2 * AT + 64), ("out", 5 * AT), ("residual_out", 3 * AT + 32),
        ("out", 4 * AT)],
    "resident_quantize_rows": [
        ("x", 0), ("out", 0), ("scales", 0), ("x", AT + 1), ("scales", 3 * AT + 2), ("xs", -1), ("os", -1), ("os", 511), ("rows", -1), ("columns", 0),
        ("columns", (1 << 30) + 1), ("dtype", 1), ("dtype", 8), ("out", AT), ("out", AT + 4000), ("scales", AT), ("scales", 2 * AT + 8)],
    "resident_int8_linear": [
        ("x", 0), ("weight", 0), ("weight_scales", 0), ("out", 0), ("x", AT + 1), ("weight", 2 * AT + 8), ("weight_scales", 3 * AT + 2),
        ("bias", 4 * AT + 1), ("out", 5 * AT + 1), ("workspace", 0), ("workspace", FAR + 8), ("workspace_bytes", 64), ("workspace_bytes", -1),
        ("xs", -1), ("ws", -512), ("ws", 520), ("ws", (1 << 22) + 16), ("os", -1), ("os", 255), ("tokens", -1), ("inner", 0), ("inner", 504),
        ("inner", 1 << 17), ("outer", 0), ("x_bytes", 1), ("x_bytes", 3), ("out_bytes", 1), ("tokens", 2**31 - 1),
        ("out", AT + 16), ("out", 2 * AT + 4096), ("out", 3 * AT), ("out", 4 * AT + 2)],
}
GIVEN = dict(x_bytes=1, x_scales=6 * AT, workspace=0, workspace_bytes=0)  # rows in 8 bits


def record(name, **changed):
    layout, fields, _ = ENTRIES[name]
    return layout.pack(*{**fields, **changed}.values())


def test_records_match_the_header(tmp_path):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no host compiler")
    lines = [f'  std::printf("%zu\\n", sizeof({struct}));' for _, _, struct in ENTRIES.values()]
    source = tmp_path / "sizes.cpp"
    source.write_text('#include <cstdio>\n#include "resident_epoch.h"\nint main() {\n' + "\n".join(lines) + "\n}\n")
    subprocess.run([compiler, f"-I{HEADER.parent}", str(source), "-o", str(tmp_path / "sizes")], check=True)
    sizes = [int(x) for x in subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.split()]
    assert sizes == [layout.size for layout, _, _ in ENTRIES.values()]


@pytest.mark.parametrize("name", list(ENTRIES))
def test_record_order_matches_the_header(name):
    """The test's own records list the header's fields in the header's order."""
    layout, fields, struct = ENTRIES[name]
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)

    def count(struct):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct, struct), text, re.S).group(1)
        n = 0
        for line in filter(None, (x.strip() for x in body.split(";"))):
            nested = re.match(r"(ResidentKv\w+) ", line)
            if nested:
                n += count(nested.group(1))
                continue
            for part in line.split(","):
                array = re.search(r"\[(\d)\]", part)
                n += int(array.group(1)) if array else 1
        return n

    assert count(struct) == len(fields) == len(layout.unpack(bytes(layout.size)))


@pytest.mark.parametrize("name,field,value", [(n, f, v) for n, bad in BAD.items() for f, v in bad])
def test_refused(lib, name, field, value):
    assert getattr(lib, name)(record(name, **{field: value}), None) == -1


@pytest.mark.parametrize("changed", [dict(x=AT + 8), dict(xs=520), dict(xs=(1 << 22) + 16), dict(x_scales=0), dict(x_scales=6 * AT + 2),
                                     dict(out=6 * AT), dict(weight=5 * AT + 64)])
def test_given_rows_are_refused(lib, changed):
    """Rows in 8 bits start at multiples of 16 bytes and bring their scales."""
    assert lib.resident_int8_linear_workspace(record("resident_int8_linear", **GIVEN)) == 0
    assert lib.resident_int8_linear(record("resident_int8_linear", **{**GIVEN, **changed}), None) == -1


@pytest.mark.parametrize("changed", [dict(out_scales=7 * AT + 16), dict(out_scales=6 * AT), dict(out_scales=AT), dict(out=AT), dict(out=2 * AT),
                                     dict(out=4 * AT, gs0=512)])
def test_norms_to_8_bits_lie_apart(lib, changed):
    """Bytes take the place of no input, nor do the scales."""
    assert lib.resident_block_norms(record("resident_block_norms", **{"out_scales": 8 * AT, **changed}), None) == -1


@pytest.mark.parametrize("changed", [dict(x=0), dict(x=0, residual_out=0), dict(x=0, residual_out=0, post_norm=0), dict(x=0, residual_out=0, gate=0)])
def test_what_needs_x(lib, changed):
    assert lib.resident_block_norms(record("resident_block_norms", **changed), None) == -1


@pytest.mark.parametrize("name", list(ENTRIES))
def test_null_record_is_refused(lib, name):
    assert getattr(lib, name)(None, None) == -1
    if name + "_workspace" in _lib.SIGNATURES:
        assert getattr(lib, name + "_workspace")(None) == -1


@pytest.mark.parametrize("name,none", [("resident_kv_prefix_attention", "rows"), ("resident_block_norms", "tokens"),
                                       ("resident_quantize_rows", "rows"), ("resident_int8_linear", "tokens")])
def test_nothing_to_do_is_done(lib, name, none):
    """No rows or tokens: accepted, nothing queued (so also without a GPU)."""
    assert getattr(lib, name)(record(name, **{none: 0}), None) == 0


def test_prefixes_longer_than_the_kernels_count(lib):
    long = dict(block=1 << 20, pages=8, prefix_width=1 << 11, kv_heads=1, ks2=64, heads=4)
    size = lib.resident_kv_prefix_attention_workspace
    assert size(record("resident_kv_prefix_attention", **long, max_prefix=1 << 30)) > 0
    assert size(record("resident_kv_prefix_attention", **long, max_prefix=(1 << 30) + 1)) == -1
    assert lib.resident_kv_prefix_attention(record("resident_kv_prefix_attention", **long, max_prefix=2**31 - 1), None) == -1


@pytest.mark.parametrize("name,changed", [("resident_kv_prefix_attention", {}), ("resident_kv_prefix_attention", dict(rows=40)),
                                          ("resident_int8_linear", {}), ("resident_int8_linear", dict(tokens=300, out=FAR))])
def test_workspace_sizes(lib, name, changed):
    if name == "resident_int8_linear" and changed:
        changed = dict(changed, workspace=2 * FAR)
    need = getattr(lib, name + "_workspace")(record(name, **changed))
    assert need > 0
    assert getattr(lib, name)(record(name, **changed, workspace_bytes=need - 1), None) == -1


def test_strides_of_single_extents_do_not_matter(lib):
    size = lib.resident_int8_linear_workspace
    assert size(record("resident_int8_linear", tokens=1, xs=3, os=1)) > 0
    assert size(record("resident_int8_linear", **GIVEN, tokens=1, xs=7)) == 0
    assert size(record("resident_int8_linear", **GIVEN, outer=1, ws=5)) == 0
    assert lib.resident_kv_prefix_attention_workspace(record("resident_kv_prefix_attention", rows=1, qs0=3, os0=5)) > 0


def test_python_refuses_what_does_not_fit():
    cache, x, i = torch.zeros(2, 16, 2, 64), torch.zeros(1, 2, 64), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="key_cache must be a tensor on a GPU"):
        ops.kv_prefix_attention(x, cache, cache, i, i, i[None], i)
    with pytest.raises(ValueError, match="residual must be a tensor on a GPU"):
        ops.block_norms(torch.zeros(1, 8), torch.zeros(1, 8), pre_norm=torch.zeros(8))
    with pytest.raises(ValueError, match="x must be a tensor on a GPU"):
        ops.quantize_rows(torch.zeros(1, 8))
    with pytest.raises(ValueError, match="x must be a tensor on a GPU"):
        ops.int8_linear(torch.zeros(1, 16), torch.zeros(2, 16, dtype=torch.int8), torch.zeros(2))
