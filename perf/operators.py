"""The serving operators over a bounded paged cache, as cases a timer can run.

Each case is one call of one operator, as a decode loop makes it:

  write   ``kv_write``: the queries and keys of new tokens are normalised for
          each head and rotated, keys and values go to their cache slots
  attend  ``kv_attention``: one new token of every row over its cached
          positions, in some cases adding each position's attention weight to
          the cache's weights
  evict   ``kv_evict``: every KV head of a row keeps its ``budget`` slots of
          greatest accumulated weight, compacted to the row's front
  logits  ``process_logits``: penalties of repeated tokens, biases and a grammar
          mask on the logits, and the greedy token of what is left

``run`` computes the plain form in elementary torch operations, or, where
``own`` is set, makes the calls of ``cruise_amd.ops``.  The shapes are this
repository's (28 query heads over 4 KV heads of 128 in bf16, pages of 128, a
vocabulary of 152,064; the tiny fp32 model's 4 over 2 heads of 64, pages of 16)
and generic ones.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
NEG_INF = float("-inf")


def listed():
    qwen = dict(heads=28, kv_heads=4, head_dim=128, block=128, dtype="bf16")
    tiny = dict(heads=4, kv_heads=2, head_dim=64, dtype="fp32")
    return [
        # One decode step of the headline batch: four tokens, latency counts.
        dict(name="write-step-4", op="write", tokens=4, far=256, norm=True, skip=0, **qwen),
        # The prompts of a 64-row batch, 1,000 tokens each.
        dict(name="write-prompts-64x1000", op="write", tokens=64000, far=1000, norm=True, skip=0, **qwen),
        # fp32, an odd count, positions far beyond a first window, some tokens not stored.
        dict(name="write-fp32-4097", op="write", tokens=4097, far=1000000, norm=False, skip=13, block=16, **tiny),
        # The headline batch at its window of 256 positions.
        dict(name="attend-step-4x256", op="attend", rows=4, length=256, lengths="ragged", weights=False, **qwen),
        # 64 rows of about 1,000 positions, their weights kept for eviction.
        dict(name="attend-64x1000", op="attend", rows=64, length=1000, lengths="ragged", weights=True, **qwen),
        # One long conversation: few rows, the cache's length is all the parallelism.
        dict(name="attend-1x131071", op="attend", rows=1, length=131071, lengths="equal", weights=False, **qwen),
        # fp32, pages that end inside every tile, empty rows, weights kept.
        dict(name="attend-fp32-12x4097", op="attend", rows=12, length=4097, lengths="empty", weights=True, block=24, **tiny),
        # A serving batch at its budget: each row is one page over it.
        dict(name="evict-16x1152", op="evict", rows=16, length=1152, budget=1024, recent=256, sinks=4, lengths="equal", **qwen),
        # Long prompts cut to a budget before decoding starts.
        dict(name="evict-8x32768", op="evict", rows=8, length=32768, budget=4096, recent=512, sinks=0, lengths="ragged", **qwen),
        # One decode step of the headline batch, all that the operator does.
        dict(name="logits-4", op="logits", rows=4, vocab=152064, history=256, biases=8, mask=True, dtype="fp32"),
        # 64 rows with long histories.
        dict(name="logits-64x8192", op="logits", rows=64, vocab=152064, history=8192, biases=16, mask=True, dtype="fp32"),
        # A small odd vocabulary in bf16, without a grammar.
        dict(name="logits-bf16-33", op="logits", rows=33, vocab=4093, history=31, biases=0, mask=False, dtype="bf16"),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["write", "attend", "evict", "logits"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "logits":
        return dict(op=op, rows=_log_uniform(rng, 1, 64), vocab=_log_uniform(rng, 1000, 152064), history=_log_uniform(rng, 1, 8192),
                    biases=rng.randint(0, 32), mask=rng.random() < 0.7, dtype=dtype)
    heads, kv_heads, head_dim = rng.choice([(28, 4, 128), (4, 2, 64), (8, 8, 64), (32, 2, 128), (16, 1, 256), (5, 5, 128), (9, 3, 256)])
    block = rng.choice([1, 16, 24, 100, 128, 256])
    shape = dict(heads=heads, kv_heads=kv_heads, head_dim=head_dim, block=block, dtype=dtype)
    # No drawn case costs more than the largest listed one: 262,144 slots of 4 x 128 bf16.
    most = 262144 * 4 * 128 * 2 // (kv_heads * head_dim * (2 if dtype == "bf16" else 4))
    if op == "write":
        return dict(op=op, tokens=_log_uniform(rng, 1, 16000), far=_log_uniform(rng, 16, 1000000), norm=rng.random() < 0.5,
                    skip=rng.choice([0, 0, 7]), **shape)
    if op == "attend":
        rows = _log_uniform(rng, 1, 64)
        return dict(op=op, rows=rows, length=_log_uniform(rng, 1, max(1, min(131072, most // 2 // rows))),
                    lengths=rng.choice(["equal", "ragged", "empty"]), weights=rng.random() < 0.5, **shape)
    rows = _log_uniform(rng, 1, 64)
    length = _log_uniform(rng, 16, min(65536, max(64, most // 4 // rows)))
    budget = _log_uniform(rng, 8, length)
    return dict(op=op, rows=rows, length=length, budget=budget, recent=rng.randint(0, budget // 2), sinks=rng.choice([0, 1, 4]),
                lengths=rng.choice(["equal", "ragged", "empty"]), **shape)


def _lengths(case, gen):
    """Positions of every row: all of them, between half and all, or every third row empty."""
    rows, n = case["rows"], case["length"]
    full = torch.full((rows,), n, dtype=torch.int32, device="cuda")
    if case["lengths"] == "equal":
        return full
    got = torch.randint((n + 1) // 2, n + 1, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    got[0] = n
    if case["lengths"] == "empty":
        got[1::3] = 0
    return got


def _pool(case, gen):
    """Key and value caches with every row's pages in random order."""
    per_row = -(-case["length"] // case["block"])
    pages = case["rows"] * per_row
    shape = (pages, case["block"], case["kv_heads"], case["head_dim"])
    dtype = DTYPES[case["dtype"]]
    keys = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)
    values = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)
    table = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).view(case["rows"], per_row)
    return keys, values, table


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    prepared = {"write": _prepare_write, "attend": _prepare_attend, "evict": _prepare_evict, "logits": _prepare_logits}[case["op"]](case, gen)
    prepared["case"] = case
    return prepared


def _prepare_write(case, gen):
    tokens, heads, kv_heads, d, block = (case[k] for k in ("tokens", "heads", "kv_heads", "head_dim", "block"))
    dtype = DTYPES[case["dtype"]]
    # The projection's output: q, k and v of a token side by side, read in place.
    qkv = torch.randn(tokens, (heads + 2 * kv_heads) * d, generator=gen, device="cuda").to(dtype)
    q, k, v = qkv.split([heads * d, kv_heads * d, kv_heads * d], dim=1)
    pages = -(-tokens // block) + 1
    slots = torch.randperm(pages * block, generator=gen, device="cuda")[:tokens].to(torch.int32)
    if case["skip"]:
        slots[:: case["skip"]] = -1
    cache = (pages, block, kv_heads, d)
    return dict(
        q=q.unflatten(1, (heads, d)), k=k.unflatten(1, (kv_heads, d)), v=v.unflatten(1, (kv_heads, d)),
        positions=torch.randint(0, case["far"], (tokens,), generator=gen, device="cuda"), slots=slots,
        q_norm=(1 + 0.1 * torch.randn(d, generator=gen, device="cuda")).to(dtype) if case["norm"] else None,
        k_norm=(1 + 0.1 * torch.randn(d, generator=gen, device="cuda")).to(dtype) if case["norm"] else None,
        inv_freq=(1e6 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)).float(),
        keys=torch.zeros(cache, dtype=dtype, device="cuda"), values=torch.zeros(cache, dtype=dtype, device="cuda"),
        weights=torch.ones(pages, kv_heads, block, device="cuda"),
        slot_positions=torch.full((pages, kv_heads, block), -1, dtype=torch.int32, device="cuda"),
    )


def _prepare_attend(case, gen):
    keys, values, table = _pool(case, gen)
    # Scores of standard deviation 2: some positions matter and most do not.
    q = 2 * torch.randn(case["rows"], case["heads"], case["head_dim"], generator=gen, device="cuda")
    got = dict(q=q.to(DTYPES[case["dtype"]]), keys=keys, values=values, table=table, lengths=_lengths(case, gen))
    if case["weights"]:
        # What the steps before have added; every pass starts from it.
        got["before"] = torch.rand(keys.shape[0], case["kv_heads"], case["block"], generator=gen, device="cuda")
        got["weights"] = got["before"].clone()
    return got


def _prepare_evict(case, gen):
    keys, values, table = _pool(case, gen)
    lengths = _lengths(case, gen)
    rows, per_row = table.shape
    kv_heads, block = case["kv_heads"], case["block"]
    # A long-tailed sum for every slot, and the token that it holds: in order, as a prompt leaves them.
    before = torch.rand(keys.shape[0], kv_heads, block, generator=gen, device="cuda").pow(-0.5) - 1
    order = torch.arange(per_row * block, dtype=torch.int32, device="cuda").view(1, per_row, 1, block)
    positions = torch.empty_like(before, dtype=torch.int32)
    positions[table.long().flatten()] = order.expand(rows, per_row, kv_heads, block).flatten(0, 1)
    return dict(keys=keys, values=values, table=table, lengths=lengths, next_positions=lengths.long(), before=before,
                weights=before.clone(), positions_before=positions, slot_positions=positions.clone())


def _prepare_logits(case, gen):
    rows, vocab, history, biases = (case[k] for k in ("rows", "vocab", "history", "biases"))
    logits = (3 * torch.randn(rows, vocab, generator=gen, device="cuda")).to(DTYPES[case["dtype"]])
    # Frequent tokens come again and again, as in text.
    ids = (vocab * torch.rand(rows, history, generator=gen, device="cuda").pow(4)).long().clamp_(max=vocab - 1)
    lengths = torch.randint((history + 1) // 2, history + 1, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    uniform = lambda low, high: low + (high - low) * torch.rand(rows, generator=gen, device="cuda")  # noqa: E731
    got = dict(logits=logits, history=ids, history_lengths=lengths, prompt_lengths=lengths // 3, repetition=uniform(1.0, 1.5),
               presence=uniform(0.0, 0.5), frequency=uniform(0.0, 0.3), bias_ids=None, bias_values=None, allowed=None)
    if biases:
        first = torch.randint(0, vocab, (rows, 1), generator=gen, device="cuda")
        got["bias_ids"] = (first + (vocab // (biases + 1)) * torch.arange(biases, device="cuda")) % vocab
        got["bias_values"] = 4 * torch.randn(rows, biases, generator=gen, device="cuda")
    if case["mask"]:
        # Half of the rows inside a grammar that allows an eighth of the vocabulary, half of them free.
        words = torch.randint(-(1 << 31), 1 << 31, (4, rows, -(-vocab // 32)), generator=gen, device="cuda")
        allowed = words[0] & words[1] & words[2]
        allowed[1::2] = -1
        got["allowed"] = allowed.to(torch.int32)
    return got


def run(state):
    return {"write": _run_write, "attend": _run_attend, "evict": _run_evict, "logits": _run_logits}[state["case"]["op"]](state)


def _run_write(s):
    if own:
        from cruise_amd import ops

        q_out = ops.kv_write(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["keys"], s["values"], s["inv_freq"],
                             q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6, weight_cache=s["weights"],
                             position_cache=s["slot_positions"])
    else:
        # Angles of far positions need 64 bits: a 32-bit product is off by up to pos * 2^-24.
        angle = s["positions"].double()[:, None] * s["inv_freq"].double()
        cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
        q_out = _plain_rotate(s["q"], s["q_norm"], cos, sin)
        k_out = _plain_rotate(s["k"], s["k_norm"], cos, sin)
        stored = s["slots"] >= 0
        slots = s["slots"][stored].long()
        block = s["keys"].shape[1]
        s["keys"].flatten(0, 1)[slots] = k_out[stored]
        s["values"].flatten(0, 1)[slots] = s["v"][stored]
        s["weights"][slots // block, :, slots % block] = 0.0
        s["slot_positions"][slots // block, :, slots % block] = s["positions"][stored].int()[:, None]
    return q_out, s["keys"], s["values"], s["weights"], s["slot_positions"]


def _plain_rotate(x, weight, cos, sin):
    n = x.float()
    if weight is not None:
        n = n * torch.rsqrt(n.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
    a, b = n.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1).to(x.dtype)


def _run_attend(s):
    weights = s.get("weights")
    if weights is not None:
        weights.copy_(s["before"])
    if own:
        from cruise_amd import ops

        out = ops.kv_attention(s["q"], s["keys"], s["values"], s["table"], s["lengths"], weight_cache=weights,
                               max_length=s["case"]["length"])
    else:
        rows, heads, d = s["q"].shape
        pages, block, kv_heads, _ = s["keys"].shape
        n = s["case"]["length"]
        at = torch.arange(n, device="cuda")
        page, offset = s["table"].long()[:, at // block], at % block
        valid = (at < s["lengths"][:, None])[:, None, None]
        k = s["keys"][page, offset].float().permute(0, 2, 1, 3)
        v = s["values"][page, offset].float().permute(0, 2, 1, 3)
        q = s["q"].float().view(rows, kv_heads, heads // kv_heads, d)
        scores = torch.where(valid, (q @ k.transpose(2, 3)) * d**-0.5, NEG_INF)
        p = torch.where(valid, (scores - scores.amax(-1, keepdim=True)).exp(), 0.0)
        p = p / torch.where(valid[..., :1], p.sum(-1, keepdim=True), 1.0)
        out = (p @ v).view(rows, heads, d).to(s["q"].dtype)
        if weights is not None:
            slot = (page[:, None] * kv_heads + torch.arange(kv_heads, device="cuda")[:, None]) * block + offset
            weights.view(-1).index_add_(0, slot.flatten(), p.sum(2).flatten())
    return (out,) if weights is None else (out, weights)


def _run_evict(s):
    case = s["case"]
    # The moved slots' keys and values stay where they came from, so these two make the pass the same again.
    s["weights"].copy_(s["before"])
    s["slot_positions"].copy_(s["positions_before"])
    if own:
        from cruise_amd import ops

        lengths = ops.kv_evict(s["keys"], s["values"], s["table"], s["lengths"], s["next_positions"], s["weights"],
                               s["slot_positions"], budget=case["budget"], recent=case["recent"], sinks=case["sinks"],
                               max_length=case["length"])
    else:
        lengths = _plain_evict(s, case)
    return s["keys"], s["values"], s["weights"], s["slot_positions"], lengths


def _plain_evict(s, case):
    block, kv_heads, budget = case["block"], case["kv_heads"], min(case["budget"], case["length"])
    at = torch.arange(case["length"], device="cuda")
    # [rows, KV heads, length]: where a slot's weight lies, and the slot's place among the cached keys
    page = s["table"].long()[:, None, at // block]
    head, offset = torch.arange(kv_heads, device="cuda")[:, None], (at % block)[None, None]
    valid = (at < s["lengths"][:, None])[:, None]
    weight, position = s["weights"][page, head, offset], s["slot_positions"][page, head, offset]
    recent = position >= s["next_positions"][:, None, None] - case["recent"]
    kept_first = (position >= 0) & (recent | (position < case["sinks"]))
    order = torch.where(valid, weight, NEG_INF).argsort(dim=-1, descending=True, stable=True)
    rank = torch.where(kept_first, 2, 1) * valid
    order = order.gather(-1, rank.gather(-1, order).argsort(dim=-1, descending=True, stable=True))
    kept = torch.zeros_like(weight, dtype=torch.bool).scatter_(-1, order[..., :budget], True) & valid
    holes = (at < budget) & ~kept & valid
    r, h, to = holes.nonzero(as_tuple=True)
    _, _, source = (kept & (at >= budget)).nonzero(as_tuple=True)
    table = s["table"].long()
    to = (table[r, to // block], to % block)
    source = (table[r, source // block], source % block)
    s["keys"][to[0], to[1], h] = s["keys"][source[0], source[1], h]
    s["values"][to[0], to[1], h] = s["values"][source[0], source[1], h]
    s["weights"][to[0], h, to[1]] = s["weights"][source[0], h, source[1]]
    s["slot_positions"][to[0], h, to[1]] = s["slot_positions"][source[0], h, source[1]]
    r, h, behind = (valid & (at >= budget)).expand(-1, kv_heads, -1).nonzero(as_tuple=True)
    s["weights"][table[r, behind // block], h, behind % block] = 0.0
    s["slot_positions"][table[r, behind // block], h, behind % block] = -1
    return s["lengths"].clamp(max=budget)


def _run_logits(s):
    names = ("history", "history_lengths", "prompt_lengths", "repetition", "presence", "frequency", "bias_ids", "bias_values", "allowed")
    if own:
        from cruise_amd import ops

        return ops.process_logits(s["logits"], **{k: s[k] for k in names})
    history, lengths, prompts, repetition, presence, frequency, bias_ids, bias_values, allowed = (s[k] for k in names)
    x = s["logits"].float()
    rows, vocab = x.shape
    at = torch.arange(history.shape[1], device="cuda")
    used = at < lengths[:, None]
    seen = torch.zeros_like(x).scatter_add_(1, history, used.float())
    count = torch.zeros_like(x).scatter_add_(1, history, (used & (at >= prompts[:, None])).float())
    x = torch.where(seen > 0, torch.where(x > 0, x / repetition[:, None], x * repetition[:, None]), x)
    x = torch.where(count > 0, x - frequency[:, None] * count - presence[:, None], x)
    if bias_ids is not None:
        x = x.scatter_add(1, bias_ids, bias_values)
    if allowed is not None:
        bits = (allowed[:, :, None] >> torch.arange(32, dtype=torch.int32, device="cuda")) & 1
        x = torch.where(bits.flatten(1)[:, :vocab] == 1, x, NEG_INF)
    top = x.amax(1, keepdim=True)
    first = torch.where(x == top, torch.arange(vocab, device="cuda"), vocab).amin(1)
    return x, torch.where(top[:, 0].isfinite(), first, -1)


def work(case):
    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        size = 2 if case["dtype"] == "bf16" else 4
        each = vocab * (size + 4) + (vocab // 8 if case["mask"] else 0) + case["history"] * 6 + case["biases"] * 12
        return {"bytes": rows * each, "flops": rows * vocab * 4}
    size = 2 if case["dtype"] == "bf16" else 4
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "write":
        values = case["tokens"] * (heads + 2 * kv_heads) * d
        return {"bytes": 2 * values * size + case["tokens"] * (12 + 8 * kv_heads), "flops": 10 * values}
    n, rows = case["length"], case["rows"]
    mean = n if case["lengths"] == "equal" else 0.75 * n * (2 / 3 if case["lengths"] == "empty" else 1)
    if case["op"] == "attend":
        each = 2 * mean * kv_heads * d * size + 2 * heads * d * size + (8 * mean * kv_heads if case["weights"] else 0)
        return {"bytes": int(rows * each), "flops": int(4 * rows * mean * heads * d)}
    # Slots behind the budget that stay: the recent ones, and their share of the others.
    budget, recent, sinks = case["budget"], case["recent"], case["sinks"]
    moved = 0.0
    if mean > budget:
        free = max(0, budget - recent - sinks) * max(0.0, mean - recent - budget) / max(1.0, mean - recent - sinks)
        moved = min(recent, mean - budget) + free
    return {"bytes": int(rows * kv_heads * (16 * mean + 4 * moved * d * size)), "flops": int(rows * kv_heads * 4 * mean)}


def exact(case, seed):
    """The operators from their definitions in 64 bits, row by row where that is simplest."""
    s = prepare(case, seed)
    return {"write": _exact_write, "attend": _exact_attend, "evict": _exact_evict, "logits": _exact_logits}[case["op"]](s, case)


def _exact_write(s, case):
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"][:, None].double() * s["inv_freq"].double())

    def rotated(x, weight):
        x = x.double()
        if weight is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * weight.double()
        half = x.shape[-1] // 2
        z = torch.complex(x[..., :half], x[..., half:]) * turn[:, None]
        return torch.cat([z.real, z.imag], -1)

    block = case["block"]
    keys, values, weights = s["keys"].double(), s["values"].double(), s["weights"].double()
    written = torch.nonzero(s["slots"] >= 0)[:, 0]
    page, offset = s["slots"][written].long() // block, s["slots"][written].long() % block
    keys[page, offset] = rotated(s["k"][written], s["k_norm"]) if len(written) == len(turn) else rotated(s["k"], s["k_norm"])[written]
    values[page, offset] = s["v"][written].double()
    weights[page, :, offset] = 0
    s["slot_positions"][page, :, offset] = s["positions"][written].to(torch.int32)[:, None].expand(-1, case["kv_heads"])
    return rotated(s["q"], s["q_norm"]), keys, values, weights, s["slot_positions"]


def _exact_attend(s, case):
    rows, heads, d = s["q"].shape
    block, kv_heads = case["block"], case["kv_heads"]
    out = torch.zeros(rows, heads, d, dtype=torch.float64, device="cuda")
    weights = s["before"].double() if case["weights"] else None
    for r, n in enumerate(s["lengths"].tolist()):
        if n == 0:
            continue
        used = s["table"][r, : -(-n // block)].long()
        for g in range(kv_heads):
            group = slice(g * heads // kv_heads, (g + 1) * heads // kv_heads)
            k = s["keys"][used, :, g].flatten(0, 1)[:n].double()
            v = s["values"][used, :, g].flatten(0, 1)[:n].double()
            p = torch.softmax(s["q"][r, group].double() @ k.T / math.sqrt(d), dim=-1)
            out[r, group] = p @ v
            if weights is not None:
                row = weights[used, g].flatten()
                row[:n] += p.sum(0)
                weights[used, g] = row.view(-1, block)
    return (out,) if weights is None else (out, weights)


def _exact_evict(s, case):
    """Nothing is computed: what stays, and where, is settled row by row with lists of its own."""
    block, budget, recent, sinks = (case[k] for k in ("block", "budget", "recent", "sinks"))
    lengths = []
    for r, n in enumerate(s["lengths"].tolist()):
        lengths.append(min(n, budget))
        if n <= budget:
            continue
        used = s["table"][r, : -(-n // block)].long()
        limit = int(s["next_positions"][r]) - recent
        for g in range(case["kv_heads"]):
            w, p = s["before"][used, g].flatten()[:n].tolist(), s["positions_before"][used, g].flatten()[:n].tolist()
            first = [p[j] >= 0 and (p[j] >= limit or p[j] < sinks) for j in range(n)]
            stay = set(sorted(range(n), key=lambda j: (not first[j], -w[j], j))[:budget])
            to = torch.tensor([j for j in range(budget) if j not in stay], dtype=torch.long, device="cuda")
            source = torch.tensor([j for j in range(budget, n) if j in stay], dtype=torch.long, device="cuda")
            for cache in (s["keys"], s["values"]):
                cache[used[to // block], to % block, g] = cache[used[source // block], source % block, g]
            for cache, empty in ((s["weights"], 0.0), (s["slot_positions"], -1)):
                cache[used[to // block], g, to % block] = cache[used[source // block], g, source % block]
                behind = torch.arange(budget, n, device="cuda")
                cache[used[behind // block], g, behind % block] = empty
    return (s["keys"].double(), s["values"].double(), s["weights"].double(), s["slot_positions"],
            torch.tensor(lengths, dtype=torch.int32, device="cuda"))


def _exact_logits(s, case):
    out = s["logits"].double()
    vocab = case["vocab"]
    best = []
    for r in range(case["rows"]):
        n, prompt = int(s["history_lengths"][r]), int(s["prompt_lengths"][r])
        row = out[r]
        seen = torch.unique(s["history"][r, :n])
        rep = s["repetition"][r].double()
        row[seen] = torch.where(row[seen] > 0, row[seen] / rep, row[seen] * rep)
        count = torch.bincount(s["history"][r, prompt:n], minlength=vocab).double()
        row -= s["frequency"][r].double() * count + s["presence"][r].double() * count.clamp(max=1)
        if s["bias_ids"] is not None:
            row[s["bias_ids"][r]] += s["bias_values"][r].double()
        if s["allowed"] is not None:
            word = s["allowed"][r].repeat_interleave(32)[:vocab]
            bit = torch.arange(vocab, dtype=torch.int32, device="cuda") % 32
            row[torch.bitwise_right_shift(word, bit) % 2 == 0] = NEG_INF
        best.append(int(torch.nonzero(row == row.max())[0, 0]) if bool(row.max() > NEG_INF) else -1)
    return out, torch.tensor(best, dtype=torch.int64, device="cuda")
