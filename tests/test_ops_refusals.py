"""The serving operators' records and refusals, without a GPU.

* The packed records of cruise_amd/ops.py have the sizes and field offsets that
  the C structs of include/resident_epoch.h have.
* Every argument that a C entry refuses comes back as -1 before anything is
  queued: one field of a good record is made bad at a time.  The addresses are
  never followed on the host, and nothing is launched.
* The Python entry points refuse tensors that are not on a GPU.
"""
from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from cruise_amd import _lib, build, ops

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "resident_epoch.h"
AT = 1 << 20  # an aligned address that nothing follows


@pytest.fixture(scope="module")
def lib():
    if not _lib.library_path().is_file():
        build.build()
    return _lib.load()


CACHE = dict(keys=AT, values=AT, weights=AT, positions=AT, ks0=16 * 4 * 64, ks1=4 * 64, ks2=64, vs0=16 * 4 * 64, vs1=4 * 64, vs2=64,
             ws0=64, ws1=16, ps0=64, ps1=16, pages=8, block=16, kv_heads=4, head_dim=64, dtype=2, device=-1)
WRITE = dict(CACHE, q=AT, k=AT, v=AT, q_out=AT, q_norm=AT, k_norm=0, inv_freq=AT, token_positions=AT, slots=AT, qs0=512, qs1=64, kss0=256,
             kss1=64, vss0=256, vss1=64, os0=512, os1=64, tokens=3, heads=8, eps=1e-6, reserved=0)
ATTEND = dict(CACHE, q=AT, out=AT, table=AT, lengths=AT, workspace=0, workspace_bytes=0, qs0=512, qs1=64, os0=512, os1=64, table_stride=4,
              rows=2, heads=8, width=4, max_length=64, scale=0.125, reserved=0)
EVICT = dict(CACHE, table=AT, lengths=AT, next_positions=AT, out_lengths=AT + 64, workspace=AT, workspace_bytes=1 << 30, table_stride=128,
             rows=2, width=128, max_length=2048, budget=1024, recent=8, sinks=4)
LOGITS = dict(logits=AT, out=2 * AT, tokens=AT, history=AT, history_lengths=AT, prompt_lengths=AT, repetition=AT, presence=AT, frequency=AT,
              bias_ids=AT, bias_values=AT, allowed=AT, workspace=AT, workspace_bytes=1 << 20, logits_stride=10000, out_stride=10000,
              history_stride=8, bias_id_stride=4, bias_value_stride=4, allowed_stride=320, rows=2, vocab=10000, width=8, biases=4, dtype=4,
              device=-1)
ENTRIES = {
    "resident_kv_write": (ops.KV_WRITE, WRITE),
    "resident_kv_attention": (ops.KV_ATTENTION, ATTEND),
    "resident_kv_evict": (ops.KV_EVICT, EVICT),
    "resident_logits_process": (ops.LOGITS, LOGITS),
}
BAD_CACHE = [
    ("keys", 0), ("values", 0), ("keys", AT + 8), ("values", AT + 2), ("weights", AT + 2), ("positions", AT + 1), ("ks0", 4), ("ks1", -64),
    ("ks2", 63), ("vs2", 4), ("ws0", -1), ("ps1", -16), ("pages", 0), ("pages", 1 << 30), ("block", 0), ("kv_heads", 0), ("head_dim", 32),
    ("head_dim", 96), ("dtype", 1), ("dtype", 8),
]
BAD = {
    "resident_kv_write": BAD_CACHE + [
        ("q", 0), ("k", 0), ("v", 0), ("q_out", 0), ("token_positions", 0), ("slots", 0), ("inv_freq", 0), ("q", AT + 4), ("q_norm", AT + 8),
        ("inv_freq", AT + 2), ("token_positions", AT + 4), ("slots", AT + 2), ("qs0", 2), ("qs1", 2), ("kss0", -8), ("vss1", 1), ("os0", 6),
        ("tokens", -1), ("heads", 0), ("heads", (1 << 20) + 1), ("eps", -1.0), ("eps", float("nan")), ("reserved", 1)],
    "resident_kv_attention": BAD_CACHE + [
        ("q", 0), ("out", 0), ("table", 0), ("lengths", 0), ("q", AT + 8), ("out", AT + 2), ("lengths", AT + 1), ("table", AT + 2),
        ("qs0", 4), ("os1", 12), ("table_stride", -1), ("rows", -1), ("rows", 1 << 20), ("heads", 0), ("heads", 6), ("width", -1),
        ("max_length", -1), ("workspace_bytes", -1), ("workspace", AT + 4), ("reserved", 7)],
    "resident_kv_evict": BAD_CACHE + [
        ("weights", 0), ("positions", 0), ("table", 0), ("lengths", 0), ("next_positions", 0), ("out_lengths", 0), ("out_lengths", AT),
        ("out_lengths", AT + 4), ("next_positions", AT + 4), ("table_stride", -4), ("rows", -1), ("rows", 1 << 20), ("width", -1),
        ("max_length", -1), ("budget", 0), ("budget", 11), ("recent", -1), ("sinks", -1), ("recent", 1021), ("recent", 2**31 - 1),
        ("workspace", 0), ("workspace", AT + 8), ("workspace_bytes", 16)],
    "resident_logits_process": [
        ("logits", 0), ("logits", AT + 2), ("out", AT + 4), ("out", AT + 2000), ("out", 2 * AT + 2), ("tokens", AT + 4), ("history", AT + 4),
        ("history_lengths", 0), ("bias_values", 0), ("bias_ids", AT + 4), ("allowed", AT + 1), ("rows", -1), ("rows", 1 << 30), ("vocab", 0),
        ("width", -1), ("width", 1 << 30), ("biases", -1), ("biases", 1 << 30), ("dtype", 1), ("logits_stride", -1), ("out_stride", 9999), ("history_stride", -8),
        ("bias_id_stride", -1), ("bias_value_stride", -1), ("allowed_stride", -1), ("workspace", 0), ("workspace", AT + 8),
        ("workspace_bytes", 0), ("workspace_bytes", -1)],
}


def record(name, **changed):
    layout, fields = ENTRIES[name]
    return layout.pack(*{**fields, **changed}.values())


def test_records_match_the_header(tmp_path):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no host compiler")
    structs = {"ResidentKvWrite": ops.KV_WRITE, "ResidentKvAttention": ops.KV_ATTENTION, "ResidentKvEvict": ops.KV_EVICT,
               "ResidentLogits": ops.LOGITS}
    lines = [f'  std::printf("%zu\\n", sizeof({s}));' for s in structs]
    source = tmp_path / "sizes.cpp"
    source.write_text('#include <cstdio>\n#include "resident_epoch.h"\nint main() {\n' + "\n".join(lines) + "\n}\n")
    subprocess.run([compiler, f"-I{HEADER.parent}", str(source), "-o", str(tmp_path / "sizes")], check=True)
    sizes = [int(x) for x in subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.split()]
    assert sizes == [layout.size for layout in structs.values()]


@pytest.mark.parametrize("name", list(ENTRIES))
def test_record_order_matches_the_header(name):
    """The test's own records list the header's fields in the header's order."""
    struct = {"resident_kv_write": "ResidentKvWrite", "resident_kv_attention": "ResidentKvAttention",
              "resident_kv_evict": "ResidentKvEvict", "resident_logits_process": "ResidentLogits"}[name]
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)

    def count(body):
        n = 0
        for line in filter(None, (x.strip() for x in body.split(";"))):
            if line.startswith("ResidentKvCache"):
                n += count(re.search(r"typedef struct ResidentKvCache \{(.*?)\} ResidentKvCache;", text, re.S).group(1))
                continue
            array = re.search(r"\[(\d)\]", line)
            n += int(array.group(1)) if array else line.count(",") + 1
        return n

    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct, struct), text, re.S).group(1)
    layout, fields = ENTRIES[name]
    assert count(body) == len(fields) == len(layout.unpack(bytes(layout.size)))


@pytest.mark.parametrize("name,field,value", [(n, f, v) for n, bad in BAD.items() for f, v in bad])
def test_refused(lib, name, field, value):
    assert getattr(lib, name)(record(name, **{field: value}), None) == -1


@pytest.mark.parametrize("name", list(ENTRIES))
def test_null_record_is_refused(lib, name):
    assert getattr(lib, name)(None, None) == -1
    if name != "resident_kv_write":
        assert getattr(lib, name + "_workspace")(None) == -1


@pytest.mark.parametrize("name,none", [("resident_kv_write", "tokens"), ("resident_kv_attention", "rows"), ("resident_kv_evict", "rows"),
                                       ("resident_logits_process", "rows")])
def test_nothing_to_do_is_done(lib, name, none):
    """No tokens or rows: accepted, nothing queued (so also without a GPU)."""
    assert getattr(lib, name)(record(name, **{none: 0}), None) == 0


def test_strides_of_single_extents_do_not_matter(lib):
    """A dimension of one element is never stepped over, whatever its stride."""
    size = lib.resident_kv_attention_workspace
    assert size(record("resident_kv_attention", rows=1, qs0=3, os0=5)) >= 0
    assert size(record("resident_kv_attention", rows=2, qs0=3)) == -1
    assert size(record("resident_kv_attention", kv_heads=1, ks2=3, vs2=1)) >= 0


@pytest.mark.parametrize("name", ["resident_kv_attention", "resident_kv_evict"])
def test_rows_longer_than_the_kernels_count(lib, name):
    long = dict(block=1 << 20, pages=8, width=1 << 11, table_stride=1 << 11, rows=1, kv_heads=1, ks2=64, heads=4)
    long = {k: v for k, v in long.items() if k in ENTRIES[name][1]}
    assert getattr(lib, name + "_workspace")(record(name, **long, max_length=1 << 30)) >= 0
    assert getattr(lib, name + "_workspace")(record(name, **long, max_length=(1 << 30) + 1)) == -1
    assert getattr(lib, name)(record(name, **long, max_length=2**31 - 1), None) == -1


def test_workspace_sizes(lib):
    need = lib.resident_kv_evict_workspace(record("resident_kv_evict"))
    assert need > 0
    assert getattr(lib, "resident_kv_evict")(record("resident_kv_evict", workspace_bytes=need - 1), None) == -1
    # a budget that no row can pass needs none
    assert lib.resident_kv_evict_workspace(record("resident_kv_evict", budget=2048)) == 0
    need = lib.resident_logits_process_workspace(record("resident_logits_process"))
    assert need > 0
    assert lib.resident_logits_process(record("resident_logits_process", workspace_bytes=need - 1), None) == -1


def test_python_refuses_tensors_off_the_gpu():
    cache = torch.zeros(2, 16, 2, 64)
    x, i = torch.zeros(1, 2, 64), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="key_cache must be a tensor on a GPU"):
        ops.kv_write(x, x, x, i.long(), i, cache, cache, torch.zeros(32))
    with pytest.raises(ValueError, match="key_cache must be a tensor on a GPU"):
        ops.kv_attention(x, cache, cache, i[None], i)
    with pytest.raises(ValueError, match="key_cache must be a tensor on a GPU"):
        ops.kv_evict(cache, cache, i[None], i, i.long(), None, None, budget=1, recent=0)
    with pytest.raises(ValueError, match="logits must be a tensor on a GPU"):
        ops.process_logits(torch.zeros(1, 8))
