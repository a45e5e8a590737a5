"""The operators of a layer's step around a caller's paged cache, as cases a timer can run.

Each case is what a decode or prefill loop does between two cache writes:

  prefix  ``kv_prefix_attention``: one new token of every row over a prefix that
          all rows share and over the row's own slots, in some cases adding the
          own slots' attention weights to the cache's weights
  linear  ``int8_linear``: rows of activations to 8 bits with a scale for each
          token, their product with 8-bit weights that have a scale for each
          channel, both scales, the bias
  norms   ``block_norms``: the norm after a block, its gate and residual scale,
          the residual sum and the norm before the next block
  normed  the two together, as a layer begins: the norm before the projection
          leaves in 8 bits, and the projection takes it as it is

``run`` computes the plain form in elementary torch operations, or, where
``own`` is set, makes the calls of ``cruise_amd.ops``.  The shapes are this
repository's (hidden size 3,584, 28 query heads over 4 KV heads of 128, an
intermediate size of 18,944, bf16, pages of 128; the tiny fp32 model's 4 over 2
heads of 64, pages of 16) and generic ones.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
NEG_INF = float("-inf")
EPS = 1e-6


def listed():
    qwen = dict(heads=28, kv_heads=4, head_dim=128, block=128, dtype="bf16")
    tiny = dict(heads=4, kv_heads=2, head_dim=64, dtype="fp32")
    return [
        # The headline batch behind a system prompt, a few dozen tokens into its answers: latency counts.
        dict(name="prefix-4x2048+64", op="prefix", rows=4, prefix=2048, length=64, lengths="ragged", weights=False, **qwen),
        # Sixteen questions about one long document: the prefix's bytes are all the work.
        dict(name="prefix-16x131071+200", op="prefix", rows=16, prefix=131071, length=200, lengths="equal", weights=False, **qwen),
        # 64 rows behind a long prefix: enough queries for the matrix cores; the own slots' weights are kept for eviction.
        dict(name="prefix-64x32768+1000", op="prefix", rows=64, prefix=32768, length=1000, lengths="ragged", weights=True, **qwen),
        # fp32, pages that end inside every tile, rows that have nothing but the prefix.
        dict(name="prefix-fp32-12x4097+333", op="prefix", rows=12, prefix=4097, length=333, lengths="empty", weights=True, block=24, **tiny),
        # The headline batch's gate projection: four tokens, the weights' bytes are all the work.
        dict(name="linear-4x3584-18944", op="linear", tokens=4, inner=3584, outer=18944, bias=False, dtype="bf16"),
        # The down projection of a 64-row batch: few channels, a long sum.
        dict(name="linear-64x18944-3584", op="linear", tokens=64, inner=18944, outer=3584, bias=False, dtype="bf16"),
        # A prefill's gate projection: a matrix product bound by the matrix cores.
        dict(name="linear-4096x3584-18944", op="linear", tokens=4096, inner=3584, outer=18944, bias=False, dtype="bf16"),
        # fp32 activations, odd counts of tokens and channels, a sum that ends inside a tile.
        dict(name="linear-fp32-333x1104-1001", op="linear", tokens=333, inner=1104, outer=1001, bias=True, dtype="fp32"),
        # One layer's norms of the headline batch: latency counts.
        dict(name="norms-4x3584", op="norms", tokens=4, hidden=3584, post=True, gate="channel", scale=1.0, dtype="bf16"),
        # The prompts of a 64-row batch, 1,000 tokens each, gated for each token and channel.
        dict(name="norms-64000x3584", op="norms", tokens=64000, hidden=3584, post=True, gate="element", scale=0.5, dtype="bf16"),
        # fp32, odd counts, rows that start at odd multiples of four bytes; no norm after the block.
        dict(name="norms-fp32-4097x1001", op="norms", tokens=4097, hidden=1001, post=False, gate="token", scale=1.0, dtype="fp32"),
        # The start of a layer at 1,000 tokens: norms to 8 bits, then the q, k and v projection with its bias.
        dict(name="normed-1000x3584-4608", op="normed", tokens=1000, hidden=3584, outer=4608, post=True, gate="channel", scale=1.0, bias=True,
             dtype="bf16"),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["prefix", "linear", "norms", "normed"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "prefix":
        heads, kv_heads, head_dim = rng.choice([(28, 4, 128), (4, 2, 64), (8, 8, 64), (32, 2, 128), (16, 1, 256), (5, 5, 128), (9, 3, 256)])
        rows = _log_uniform(rng, 1, 64)
        # No drawn case costs more than the largest listed one, in bytes or in products (fp32's run at a sixteenth of bf16's rate).
        slots = min(131072, 131072 * 4 * 128 * 2 // (kv_heads * head_dim * (2 if dtype == "bf16" else 4)),
                    64 * 28 * 128 * 32768 // (rows * heads * head_dim * (1 if dtype == "bf16" else 16)))
        return dict(op=op, rows=rows, prefix=_log_uniform(rng, 1, max(1, slots)), length=_log_uniform(rng, 1, min(4096, max(1, slots // rows))),
                    lengths=rng.choice(["equal", "ragged", "empty"]), weights=rng.random() < 0.5, heads=heads, kv_heads=kv_heads,
                    head_dim=head_dim, block=rng.choice([1, 16, 24, 100, 128, 256]), dtype=dtype)
    if op == "norms":
        hidden = _log_uniform(rng, 64, 18944)
        return dict(op=op, tokens=_log_uniform(rng, 1, max(1, min(64000, 64000 * 3584 // hidden // (1 if dtype == "bf16" else 2)))), hidden=hidden,
                    post=rng.random() < 0.5, gate=rng.choice(["none", "channel", "token", "element"]), scale=rng.choice([1.0, 0.5, 0.22]),
                    dtype=dtype)
    # (What the norms leave is next to a border between two steps now and then, and either is right; half-width sums of
    # hundreds of values are what that does not show in.)
    inner, outer = 16 * _log_uniform(rng, 4 if op == "linear" else 32, 1184), _log_uniform(rng, 1, 18944)
    tokens = _log_uniform(rng, 1, max(1, min(8192, 4096 * 3584 * 18944 // (inner * outer), 64000 * 3584 // inner)))
    case = dict(op=op, tokens=tokens, outer=outer, bias=rng.random() < 0.5, dtype=dtype if op == "linear" else "bf16")
    if op == "linear":
        return dict(case, inner=inner)
    return dict(case, hidden=inner, post=rng.random() < 0.5, gate=rng.choice(["none", "channel", "token", "element"]),
                scale=rng.choice([1.0, 0.5]))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "prefix":
        prepared = _prepare_prefix(case, gen)
    else:
        prepared = {}
        if case["op"] != "linear":
            prepared.update(_prepare_norms(case, gen))
        if case["op"] != "norms":
            prepared.update(_prepare_linear(case, gen))
    prepared["case"] = case
    return prepared


def _prepare_prefix(case, gen):
    rows, n, block, kv_heads, d = (case[k] for k in ("rows", "length", "block", "kv_heads", "head_dim"))
    dtype = DTYPES[case["dtype"]]
    shared, per_row = -(-case["prefix"] // block), -(-n // block)
    pages = shared + rows * per_row
    shape = (pages, block, kv_heads, d)
    keys = torch.randn(shape, generator=gen, device="cuda").to(dtype)
    values = torch.randn(shape, generator=gen, device="cuda").to(dtype)
    # The prefix's pages and every row's lie anywhere in the pool.
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    lengths = torch.full((rows,), n, dtype=torch.int32, device="cuda")
    if case["lengths"] != "equal":
        lengths = torch.randint((n + 1) // 2, n + 1, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        lengths[0] = n
        if case["lengths"] == "empty":
            lengths[1::3] = 0
    # Scores of standard deviation 2: some positions matter and most do not.
    q = 2 * torch.randn(rows, case["heads"], d, generator=gen, device="cuda")
    got = dict(q=q.to(dtype), keys=keys, values=values, prefix_table=order[:shared].contiguous(),
               prefix_length=torch.full((1,), case["prefix"], dtype=torch.int32, device="cuda"),
               table=order[shared:].view(rows, per_row).contiguous(), lengths=lengths)
    if case["weights"]:
        # What the steps before have added; every pass starts from it.
        got["before"] = torch.rand(pages, kv_heads, block, generator=gen, device="cuda")
        got["weights"] = got["before"].clone()
    return got


def _prepare_norms(case, gen):
    tokens, hidden = case["tokens"], case["hidden"]
    dtype = DTYPES[case["dtype"]]
    randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    # A residual stream grows with the layers, and a few of its channels far more than the others; the norm's weights take those back.
    loud = 1 + 20 * (torch.rand(hidden, generator=gen, device="cuda") < 0.01)
    gate = {"none": None, "channel": (hidden,), "token": (tokens, 1), "element": (tokens, hidden)}[case["gate"]]
    return dict(block_out=randn(tokens, hidden).to(dtype), residual=(3 * loud * randn(tokens, hidden)).to(dtype),
                post_norm=(1 + 0.1 * randn(hidden)).to(dtype) if case["post"] else None,
                gate=None if gate is None else randn(*gate).tanh().to(dtype), pre_norm=((1 + 0.1 * randn(hidden)) / loud).to(dtype))


def _prepare_linear(case, gen):
    inner, outer = case.get("inner") or case["hidden"], case["outer"]
    dtype = DTYPES[case["dtype"]]
    # The weights of a program that quantised them once: the largest of a channel is 127 steps.
    w = torch.randn(outer, inner, generator=gen, device="cuda").mul_(inner**-0.5)
    weight_scale = w.abs().amax(1) / 127
    got = dict(weight=(w / weight_scale[:, None]).round_().to(torch.int8), weight_scale=weight_scale, bias=None)
    del w
    if case["bias"]:
        got["bias"] = torch.randn(outer, generator=gen, device="cuda").to(dtype)
    if case["op"] == "linear":
        loud = 1 + 10 * (torch.rand(inner, generator=gen, device="cuda") < 0.01)
        got["x"] = (loud * torch.randn(case["tokens"], inner, generator=gen, device="cuda")).to(dtype)
    return got


def run(state):
    return {"prefix": _run_prefix, "linear": _run_linear, "norms": _run_norms, "normed": _run_normed}[state["case"]["op"]](state)


def _run_prefix(s):
    case = s["case"]
    weights = s.get("weights")
    if weights is not None:
        weights.copy_(s["before"])
    if own:
        from cruise_amd import ops

        out = ops.kv_prefix_attention(s["q"], s["keys"], s["values"], s["prefix_table"], s["prefix_length"], s["table"], s["lengths"],
                                      weight_cache=weights, max_prefix=case["prefix"], max_length=case["length"])
    else:
        rows, heads, d = s["q"].shape
        _, block, kv_heads, _ = s["keys"].shape
        m, n, group = case["prefix"], case["length"], heads // kv_heads
        # The prefix, once for all rows: its KV heads' [slots, d] against the [rows * group, d] queries.
        at = torch.arange(m, device="cuda")
        page, offset = s["prefix_table"].long()[at // block], at % block
        k = s["keys"][page, offset].float().permute(1, 0, 2)
        v = s["values"][page, offset].float().permute(1, 0, 2)
        q = s["q"].float().view(rows, kv_heads, group, d)
        shared = q.permute(1, 0, 2, 3).reshape(kv_heads, rows * group, d) @ k.transpose(1, 2) * d**-0.5
        shared = shared.view(kv_heads, rows, group, m).permute(1, 0, 2, 3)
        shared = torch.where(at < s["prefix_length"], shared, NEG_INF)
        # The rows' own slots.
        at = torch.arange(n, device="cuda")
        page, offset = s["table"].long()[:, at // block], at % block
        valid = (at < s["lengths"][:, None])[:, None, None]
        k_own = s["keys"][page, offset].float().permute(0, 2, 1, 3)
        v_own = s["values"][page, offset].float().permute(0, 2, 1, 3)
        alone = torch.where(valid, q @ k_own.transpose(2, 3) * d**-0.5, NEG_INF)
        top = torch.maximum(shared.amax(-1, keepdim=True), alone.amax(-1, keepdim=True))
        shared, alone = (shared - top).exp(), (alone - top).exp()
        total = shared.sum(-1, keepdim=True) + alone.sum(-1, keepdim=True)
        out = (shared.permute(1, 0, 2, 3).reshape(kv_heads, rows * group, m) @ v).view(kv_heads, rows, group, d).permute(1, 0, 2, 3)
        out = ((out + alone @ v_own) / total).reshape(rows, heads, d).to(s["q"].dtype)
        if weights is not None:
            slot = (page[:, None] * kv_heads + torch.arange(kv_heads, device="cuda")[:, None]) * block + offset
            weights.view(-1).index_add_(0, slot.flatten(), (alone / total).sum(2).flatten())
    return (out,) if weights is None else (out, weights)


def _run_linear(s):
    if own:
        from cruise_amd import ops

        return ops.int8_linear(s["x"], s["weight"], s["weight_scale"], bias=s["bias"])
    return _plain_product(*_plain_quantise(s["x"]), s)


def _plain_quantise(x):
    x = x.float()
    scale = x.abs().amax(1) / 127
    return torch.where(scale[:, None] > 0, x / scale[:, None], 0.0).round(), scale


def _plain_product(x, x_scale, s):
    y = (x @ s["weight"].float().T) * (x_scale[:, None] * s["weight_scale"])
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(DTYPES[s["case"]["dtype"]])


def _run_norms(s):
    if own:
        from cruise_amd import ops

        return ops.block_norms(s["block_out"], s["residual"], post_norm=s["post_norm"], gate=s["gate"], scale=s["case"]["scale"],
                               pre_norm=s["pre_norm"], eps=EPS)
    dtype = s["residual"].dtype
    residual, normed = _plain_norms(s)
    return residual.to(dtype), normed.to(dtype)


def _plain_norms(s):
    n = s["block_out"].float()
    if s["post_norm"] is not None:
        n = n * torch.rsqrt(n.square().mean(1, keepdim=True) + EPS) * s["post_norm"].float()
    if s["gate"] is not None:
        n = n * s["gate"].float()
    residual = s["residual"].float() + s["case"]["scale"] * n
    return residual, residual * torch.rsqrt(residual.square().mean(1, keepdim=True) + EPS) * s["pre_norm"].float()


def _run_normed(s):
    if own:
        from cruise_amd import ops

        residual, x, x_scale = ops.block_norms(s["block_out"], s["residual"], post_norm=s["post_norm"], gate=s["gate"], scale=s["case"]["scale"],
                                               pre_norm=s["pre_norm"], eps=EPS, quantize=True)
        return residual, ops.int8_linear(x, s["weight"], s["weight_scale"], x_scale=x_scale, bias=s["bias"], dtype=residual.dtype)
    residual, normed = _plain_norms(s)
    return residual.to(s["residual"].dtype), _plain_product(*_plain_quantise(normed), s)


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "prefix":
        heads, kv_heads, d, rows, n = (case[k] for k in ("heads", "kv_heads", "head_dim", "rows", "length"))
        mean = n if case["lengths"] == "equal" else 0.75 * n * (2 / 3 if case["lengths"] == "empty" else 1)
        each = 2 * kv_heads * d * size
        nbytes = (case["prefix"] + rows * mean) * each + 2 * rows * heads * d * size + (8 * rows * mean * kv_heads if case["weights"] else 0)
        return {"bytes": int(nbytes), "flops": int(4 * rows * (case["prefix"] + mean) * heads * d)}
    tokens, nbytes, flops = case["tokens"], 0, 0
    if case["op"] != "linear":
        hidden = case["hidden"]
        gate = {"none": 0, "channel": hidden, "token": tokens, "element": tokens * hidden}[case["gate"]]
        nbytes += (3 * tokens * hidden + gate + (2 if case["post"] else 1) * hidden) * size
        flops += 12 * tokens * hidden
    if case["op"] == "norms":
        return {"bytes": nbytes + tokens * case["hidden"] * size, "flops": flops}
    inner, outer = case.get("inner") or case["hidden"], case["outer"]
    nbytes += outer * inner + 4 * outer + tokens * outer * size + (outer * size if case["bias"] else 0)
    if case["op"] == "linear":
        nbytes += tokens * inner * size
    return {"bytes": nbytes, "flops": flops + 2 * tokens * inner * outer}


def exact(case, seed):
    """The operators from their definitions in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "prefix":
        return _exact_prefix(s, case)
    if case["op"] == "linear":
        return _exact_product(s["x"].double(), s)
    residual, normed = _exact_norms(s)
    return (residual, normed) if case["op"] == "norms" else (residual, _exact_product(normed, s))


def _exact_prefix(s, case):
    """Each part's own softmax, and the two by their sums' logarithms."""
    rows, heads, d = s["q"].shape
    block, kv_heads = case["block"], case["kv_heads"]
    group = heads // kv_heads
    out = torch.zeros(rows, heads, d, dtype=torch.float64, device="cuda")
    weights = s["before"].double() if case["weights"] else None
    q = s["q"].double() / math.sqrt(d)
    shared = s["prefix_table"].long()
    for g in range(kv_heads):
        mine = slice(g * group, (g + 1) * group)
        k = s["keys"][shared, :, g].flatten(0, 1)[: case["prefix"]].double()
        v = s["values"][shared, :, g].flatten(0, 1)[: case["prefix"]].double()
        score = torch.matmul(q[:, mine].reshape(rows * group, d), k.T.contiguous())
        whole = torch.logsumexp(score, -1).view(rows, group)
        first = torch.matmul(torch.softmax(score, -1), v).view(rows, group, d)
        for r, n in enumerate(s["lengths"].tolist()):
            if n == 0:
                out[r, mine] = first[r]
                continue
            used = s["table"][r, : -(-n // block)].long()
            k = s["keys"][used, :, g].flatten(0, 1)[:n].double()
            v = s["values"][used, :, g].flatten(0, 1)[:n].double()
            score = torch.matmul(q[r, mine], k.T.contiguous())
            share = torch.sigmoid(torch.logsumexp(score, -1) - whole[r])[:, None]
            p = torch.softmax(score, -1) * share
            out[r, mine] = first[r] * (1 - share) + torch.matmul(p, v)
            if weights is not None:
                row = weights[used, g].flatten()
                row[:n] += p.sum(0)
                weights[used, g] = row.view(-1, block)
    return (out,) if weights is None else (out, weights)


def _exact_product(x, s):
    """The step of a row is an fp32 number and its values are fp32 quotients: both belong to the format."""
    step = (x.abs().max(dim=1, keepdim=True).values.float() / 127).double()
    q = torch.div(x.float().double(), step).float().double()
    q = torch.where(step == 0, torch.zeros_like(q), q).round()
    y = torch.matmul(q * step, (s["weight"].double() * s["weight_scale"].double()[:, None]).T.contiguous())
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_norms(s):
    x = s["block_out"].double()
    if s["post_norm"] is not None:
        x = x / (x.pow(2).sum(1, keepdim=True) / x.shape[1] + EPS).sqrt() * s["post_norm"].double()
    if s["gate"] is not None:
        x = x * s["gate"].double()
    r = torch.add(s["residual"].double(), x, alpha=s["case"]["scale"])
    return r, r / (r.pow(2).sum(1, keepdim=True) / r.shape[1] + EPS).sqrt() * s["pre_norm"].double()
