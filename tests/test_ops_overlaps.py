"""Which places of an output kv_write and kv_attention take, without a GPU: the
queries' own, and those apart from every row that the call reads."""
from __future__ import annotations

import pytest

from test_ops_refusals import AT, ATTEND, WRITE, lib, record  # noqa: F401  (lib: a fixture)

NO_DEVICE = 1 << 20  # accepted arguments end at the device, before any launch
D = 64  # elements of a head; bf16: two bytes each
# A projection's rows: 8 query heads, 4 key and 4 value heads.
ROW = 16 * D
QKV = dict(q=AT, k=AT + 2 * 8 * D, v=AT + 2 * 12 * D, qs0=ROW, qs1=D, kss0=ROW, kss1=D, vss0=ROW, vss1=D, keys=64 * AT, values=65 * AT)
QUERIES = dict(q=AT, qs0=ROW, qs1=D, keys=64 * AT, values=65 * AT)


def out(elements, row=ROW, head=D, **more):
    return dict(os0=row, os1=head, at=AT + 2 * elements, **more)


WIDE = {key: 2 * ROW for key in ("qs0", "kss0", "vss0")}  # rows with as much room behind them
APART = [out(0), out(10 * ROW), out(10 * ROW, 8 * D), out(-3 * ROW), out(ROW, 2 * ROW, **WIDE), out(3 * ROW, 2 * ROW, **WIDE),
         out(5 * ROW + 8 * D, 2 * ROW, **WIDE), out(-ROW, 2 * ROW, **WIDE), out(10 * ROW, D, 3 * D)]
OVER = [out(D), out(-D), out(0, 8 * D), out(ROW), out(0, ROW, 2 * D), out(0, 2 * ROW), out(0, 0), out(10 * ROW, 0), out(10 * ROW, ROW, 0),
        out(10 * ROW, 7 * D), out(10 * ROW, D, 2 * D), out(10 * ROW, ROW, D // 2), out(ROW + 12 * D, 2 * ROW, **WIDE)]


def write(lib, where, **more):  # noqa: F811
    where = dict(where)
    fields = {**QKV, **more, "q_out": where.pop("at"), **where}
    return lib.resident_kv_write(record("resident_kv_write", **fields, device=NO_DEVICE), None)


def attend(lib, where, **more):  # noqa: F811
    where = {k: v for k, v in where.items() if k in ATTEND or k == "at"}
    fields = {**QUERIES, "rows": 3, **more, "out": where.pop("at"), **where}
    return lib.resident_kv_attention_workspace(record("resident_kv_attention", **fields))


@pytest.mark.parametrize("where", APART)
def test_apart(lib, where):  # noqa: F811
    assert WRITE["tokens"] == 3 and write(lib, where) == -2
    assert attend(lib, where) >= 0


@pytest.mark.parametrize("where", OVER)
def test_over(lib, where):  # noqa: F811
    assert write(lib, where) == -1
    assert attend(lib, where) == -1


def test_over_keys_or_values(lib):  # noqa: F811
    for at in (8 * D, 4 * D, 11 * D, 15 * D, 15 * D - ROW):
        assert write(lib, out(at)) == -1
    for key in ("q", "k", "v"):  # each by itself, in storage of its own
        fields = dict(q=8 * AT, k=16 * AT, v=24 * AT)
        assert write(lib, dict(at=fields[key] + 2 * ROW, os0=ROW, os1=D), **fields) == -1
        assert write(lib, dict(at=fields[key] + 2 * 4 * ROW, os0=ROW, os1=D), **fields) == -2


def test_heads_side_by_side(lib):  # noqa: F811
    """Queries and outputs head by head: [row][head][queries, output]."""
    pairs = dict(qs0=ROW, qs1=2 * D)
    assert attend(lib, out(D, ROW, 2 * D), **pairs) >= 0
    assert attend(lib, out(D // 2, ROW, 2 * D), **pairs) == -1
    assert attend(lib, out(2 * D, ROW, 2 * D), **pairs) == -1


def test_rows_of_one(lib):  # noqa: F811
    """The stride of a single row or head is never used."""
    assert attend(lib, out(0, 8), rows=1) >= 0
    assert attend(lib, out(D, 8), rows=1) == -1
    assert write(lib, out(0, 8), tokens=1) == -2
    assert attend(lib, out(0, ROW, 8), heads=1, kv_heads=1) >= 0
    assert attend(lib, out(0, ROW, 8), heads=1, kv_heads=1, rows=1) >= 0


def test_queries_without_strides(lib):  # noqa: F811
    """Rows that share one row of queries have no place in it for their outputs."""
    shared = dict(qs0=0)
    assert attend(lib, out(0, 0), **shared) == -1
    assert attend(lib, out(0), **shared) == -1
    assert attend(lib, out(8 * D, 8 * D), **shared) >= 0
