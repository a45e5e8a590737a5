"""process_logits against its formula: bit for bit against the steps rounded to
fp32 one by one, and within their roundings of the formula in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from cruise_amd import ops
from kv_ops_reference import process_logits, wide

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def make(rows, vocab, history, biases, dtype, *, mask=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    a = dict(logits=(3 * torch.randn(rows, vocab, generator=gen)).to(dtype).cuda())
    if history:
        a["history"] = (vocab * torch.rand(rows, history, generator=gen).pow(3)).long().clamp(max=vocab - 1).cuda()
        a["history_lengths"] = torch.randint(0, history + 1, (rows,), generator=gen, dtype=torch.int32).cuda()
        a["prompt_lengths"] = (a["history_lengths"] // 2).int()
        a["repetition"] = (0.8 + torch.rand(rows, generator=gen)).cuda()
        a["presence"] = torch.randn(rows, generator=gen).cuda()
        a["frequency"] = torch.randn(rows, generator=gen).cuda()
    if biases:
        a["bias_ids"] = torch.randint(-1, vocab, (rows, biases), generator=gen).cuda()
        a["bias_values"] = (5 * torch.randn(rows, biases, generator=gen)).cuda()
    if mask:
        a["allowed"] = torch.randint(-(2**31), 2**31, (rows, (vocab + 31) // 32), generator=gen).int().cuda()
        a["allowed"][rows // 2] = -1
    return a


def run(a, **more):
    options = {k: v for k, v in a.items() if k != "logits"}
    steps, tokens = process_logits(a["logits"], np.float32, **options)
    ref, _ = process_logits(a["logits"], np.float64, **options)
    size, _ = process_logits(a["logits"].abs(), np.float64, **{
        k: (v.abs() if k == "bias_values" else -v.abs() if k in ("presence", "frequency") else v) for k, v in options.items() if k != "allowed"})
    out, got = ops.process_logits(**a, **more)
    np.testing.assert_array_equal(wide(out), steps.astype(np.float64))
    np.testing.assert_array_equal(got.cpu().numpy(), tokens)
    finite = np.isfinite(ref)
    out64, ref, size = (x[finite] for x in (wide(out), ref, size))
    # five roundings at most (quotient or product, count's product, two differences, the bias), each of the values met so far;
    # a repetition below 1 makes a quotient larger than the size's product
    bound = 5 * 2.0**-24 * (np.abs(ref) + 2 * size)
    assert (np.abs(out64 - ref) <= bound).all()
    return out, got


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab,history,biases,mask", [
    (1, 1, 1, 1, False), (3, 31, 5, 2, True), (2, 33, 40, 3, True), (5, 4096, 64, 8, True), (4, 4097, 300, 0, True), (2, 8191, 1, 1, False),
    (3, 50001, 1000, 33, True), (4, 152064, 256, 8, True), (2, 16385, 9000, 300, False), (33, 4093, 31, 0, False),
    (16, 9001, 1024, 64, True), (2, 9001, 2048, 64, True), (17, 20001, 3000, 65, False), (16, 8193, 1500, 0, True)])
def test_shapes(rows, vocab, history, biases, mask, dtype):
    run(make(rows, vocab, history, biases, dtype, mask=mask, seed=rows + vocab))


@pytest.mark.parametrize("left", ["history", "bias_ids", "allowed", "all", "prompt_lengths", "repetition", "presence", "frequency"])
def test_steps_left_out(left):
    a = make(3, 5000, 50, 4, F32, seed=1)
    gone = {"history": ("history", "history_lengths", "prompt_lengths", "repetition", "presence", "frequency"),
            "bias_ids": ("bias_ids", "bias_values"), "all": tuple(k for k in a if k != "logits")}.get(left, (left,))
    run({k: v for k, v in a.items() if k not in gone})


def test_histories_of_one_token_repeated():
    """Thousands of times the same token, counted exactly; lengths out of range are cut."""
    a = make(3, 3001, 6000, 0, F32, mask=False, seed=2)
    a["history"][0] = 2999
    a["history"][1, ::2] = 0
    a["history_lengths"] = torch.tensor([6000, 2**31 - 1, -3], dtype=torch.int32).cuda()
    a["prompt_lengths"] = torch.tensor([1, -7, 2**31 - 1], dtype=torch.int32).cuda()
    run(a)


def test_ids_out_of_range_and_repeated_biases():
    a = make(2, 700, 40, 12, F32, seed=3)
    a["history"][0, ::3], a["history"][1, ::3] = -1, 700
    a["history"][0, 1], a["history"][1, 1] = 2**62, -(2**63)
    a["history_lengths"].fill_(40)
    a["bias_ids"][0] = torch.tensor([5, 5, 699, 5, -1, 700, 2**40, 699, 6, 6, 5, 6]).cuda()
    a["allowed"].fill_(-1)
    run(a)


def test_ties_take_the_lowest_id():
    a = dict(logits=torch.zeros(4, 9001, device="cuda"))
    a["logits"][1, 4096:] = 2.0
    a["logits"][2, [8000, 17, 4095]] = 3.0
    a["logits"][3] = -0.0
    a["logits"][3, 5000] = 0.0
    assert run(a)[1].tolist() == [0, 4096, 17, 0]


def test_rows_without_a_choice():
    """Everything masked, a NaN, an infinity: -1; a masked NaN or infinity does not matter; -infinity is a masked logit."""
    a = dict(logits=torch.randn(6, 5000, device="cuda"), allowed=torch.full((6, 157), -1, dtype=torch.int32, device="cuda"))
    a["allowed"][0] = 0
    a["logits"][1, 4999] = float("nan")
    a["logits"][2, 7] = float("inf")
    a["logits"][3, 64], a["logits"][3, 65] = float("nan"), float("inf")
    a["allowed"][3, 2] = 0
    a["logits"][4] = float("-inf")
    a["logits"][5] = float("-inf")
    a["logits"][5, 4321] = -3e38
    tokens = run(a)[1].tolist()
    assert tokens[:3] == [-1, -1, -1] and tokens[3] >= 0 and tokens[4:] == [-1, 4321]


def test_in_place_and_views():
    """Rows of a wider buffer at odd addresses, written over themselves; strided parameters' rows."""
    a = make(3, 1501, 20, 6, F32, seed=4)
    want, tokens = run(a)
    wide_rows = torch.full((3, 1777), 7.0, device="cuda")
    wide_rows[:, 3:1504] = a["logits"]
    allowed = torch.zeros(3, 60, dtype=torch.int32, device="cuda")
    allowed[:, 5:52] = a["allowed"]
    history = torch.zeros(3, 31, dtype=torch.int64, device="cuda")
    history[:, 4:24] = a["history"]
    view = wide_rows[:, 3:1504]
    out, got = ops.process_logits(**{**a, "logits": view, "allowed": allowed[:, 5:52], "history": history[:, 4:24]}, out=view)
    assert out.data_ptr() == view.data_ptr() and torch.equal(out, want) and torch.equal(got, tokens)
    assert bool((wide_rows[:, :3] == 7).all()) and bool((wide_rows[:, 1504:] == 7).all())


def test_no_rows():
    out, tokens = ops.process_logits(torch.zeros(0, 9, device="cuda"))
    assert out.shape == (0, 9) and tokens.shape == (0,)


def test_graph_on_another_stream():
    a = make(4, 20000, 64, 4, F32, seed=5)
    out, tokens = torch.empty(4, 20000, device="cuda"), torch.empty(4, dtype=torch.int64, device="cuda")
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        ops.process_logits(**a, out=out, tokens=tokens)
    for step in range(4):
        a["logits"].normal_()
        a["history_lengths"].fill_(step * 20)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ref, want = process_logits(a["logits"], np.float32, **{k: v for k, v in a.items() if k != "logits"})
        np.testing.assert_array_equal(wide(out), ref.astype(np.float64))
        np.testing.assert_array_equal(tokens.cpu().numpy(), want)


def test_python_refusals():
    a = make(2, 100, 5, 3, F32)
    for name, bad in (("logits", a["logits"].half()), ("logits", a["logits"][0]), ("history", a["history"].int()), ("history_lengths", None),
                      ("history_lengths", a["history_lengths"].long()), ("prompt_lengths", a["prompt_lengths"][:1]), ("bias_values", None),
                      ("bias_values", a["bias_values"][:, :2]), ("bias_ids", a["bias_ids"].int()), ("allowed", a["allowed"][:, :3]),
                      ("repetition", a["repetition"].double()), ("logits", a["logits"].cpu()), ("logits", a["logits"].t())):
        with pytest.raises(ValueError):
            ops.process_logits(**{**a, name: bad})
    with pytest.raises(ValueError):
        ops.process_logits(a["logits"][:, :50], out=a["logits"][:, 25:75])
    with pytest.raises(ValueError):
        ops.process_logits(a["logits"], tokens=torch.zeros(2, dtype=torch.int32, device="cuda"))


def test_more_rows_than_a_record_counts():
    """As the other operators: a number that the record cannot hold is a ValueError."""
    rows = 1 << 31
    one = torch.zeros(1, 1, device="cuda")
    with pytest.raises(ValueError, match="out of range"):
        ops.process_logits(one.expand(rows, 1), out=one.expand(rows, 1))
    torch.cuda.empty_cache()
