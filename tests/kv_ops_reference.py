"""The serving operators from their definitions, in 64 bits on the CPU, slot by
slot: what the tests of cruise_amd.ops compare with."""
from __future__ import annotations

import math

import numpy as np
import torch

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}  # largest relative error of a rounding


def cpu(t):
    return t.detach().cpu()


def wide(t) -> np.ndarray:
    return cpu(t).double().numpy()


def rotated(x, norm, eps, positions, inv_freq):
    """(result, |n_1| + |n_2| of each pair): the second bounds fp32 errors."""
    n = wide(x)
    if norm is not None:
        n = n / np.sqrt((n * n).mean(-1, keepdims=True) + eps) * wide(norm)
    angle = cpu(positions).numpy().astype(np.float64)[:, None] * wide(inv_freq)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    half = n.shape[-1] // 2
    a, b = n[..., :half], n[..., half:]
    size = np.abs(a) + np.abs(b)
    return np.concatenate([a * c - b * s, b * c + a * s], -1), np.concatenate([size, size], -1)


def write_tolerance(ref, size, dtype, d):
    # The sum of d squares, the root and the products: at most d / 2 + 16 fp32
    # roundings of a pair's size; one rounding to the stored type.
    return HALF_STEP[dtype] * np.abs(ref) + (d / 2 + 16) * 2.0**-24 * size * (1 + HALF_STEP[dtype])


def slots_of(table_row, length, bound, pages, block):
    """[(page, offset)] of a row's slots; None in the place of a bad page's."""
    out = []
    for j in range(max(0, min(int(length), bound))):
        page = int(table_row[j // block])
        out.append((page, j % block) if 0 <= page < pages else None)
    return out


def attention(q, keys, values, table, lengths, scale=None, bound=None):
    """Per (row, query head): output, per-slot probabilities, and the tolerances
    of both.  Rounding points of the operator: products of stored values, sums
    and softmax in fp32, probabilities rounded to the stored type for P.V, one
    rounding of the output."""
    dtype = q.dtype
    q, k, v = wide(q), wide(keys), wide(values)
    pages, block, kv_heads, d = k.shape
    rows, heads, _ = q.shape
    scale = d**-0.5 if scale is None else scale
    bound = min(table.shape[1] * block, bound if bound is not None else 1 << 30)
    half = HALF_STEP[dtype]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    probabilities = []
    for r in range(rows):
        slots = [s for s in slots_of(cpu(table)[r], cpu(lengths)[r], bound, pages, block) if s is not None]
        per_head = []
        for h in range(heads):
            g = h // (heads // kv_heads)
            if not slots:
                per_head.append((slots, np.zeros(0), np.zeros(0)))
                continue
            at = tuple(np.array(slots).T)
            kk, vv = k[at[0], at[1], g], v[at[0], at[1], g]
            s = scale * (kk @ q[r, h])
            p = np.exp(s - s.max())
            p /= p.sum()
            # fp32 dot of d products and the scaling (errors go by the size of the scale, whatever its sign), for the
            # slot and for the maximum; then exp and the sum of p.
            delta = 2 * abs(scale) * (np.abs(kk) @ np.abs(q[r, h])).max() * (d + 4) * 2.0**-24
            delta += (len(slots) + 16) * 2.0**-24
            size = p @ np.abs(vv)
            out[r, h] = p @ vv
            tol[r, h] = half * np.abs(out[r, h]) + (half + delta) * size * (1 + half)
            per_head.append((slots, p, delta * p))
        probabilities.append(per_head)
    return out, tol, probabilities


def weights_after(before, probabilities, kv_heads):
    """The weight cache after an attention call, and its tolerance."""
    ref, tol = wide(before), 0 * wide(before)
    for per_head in probabilities:
        group = len(per_head) // kv_heads
        for h, (slots, p, dp) in enumerate(per_head):
            for (page, at), x, dx in zip(slots, p, dp):
                ref[page, h // group, at] += x
                tol[page, h // group, at] += dx + group * 2.0**-24 * x
    return ref, tol + 2.0**-24 * np.abs(ref)


def evict(keys, values, weights, positions, table, lengths, next_positions, budget, recent, sinks, bound=None):
    """New (keys, values, weights, positions, lengths); the inputs stay as they are."""
    keys, values, weights, positions = (cpu(t).clone() for t in (keys, values, weights, positions))
    table, lengths, next_positions = cpu(table), cpu(lengths), cpu(next_positions)
    pages, block, kv_heads, _ = keys.shape
    bound = min(table.shape[1] * block, bound if bound is not None else 1 << 30)
    new = []
    for r in range(table.shape[0]):
        slots = slots_of(table[r], lengths[r], bound, pages, block)
        n = len(slots)
        if None in slots or n <= budget:
            new.append(n)
            continue
        new.append(budget)
        limit = int(next_positions[r]) - recent
        for g in range(kv_heads):
            def rank(j, g=g):
                page, at = slots[j]
                w, p = float(weights[page, g, at]), int(positions[page, g, at])
                if p >= 0 and (p < sinks or p >= limit):
                    return (0, 0.0, j)
                return (1, 0.0, j) if math.isnan(w) else (2, -w + 0.0, j)

            stay = set(sorted(range(n), key=rank)[:budget])
            holes = [j for j in range(budget) if j not in stay]
            movers = [j for j in range(budget, n) if j in stay]
            assert len(holes) == len(movers)
            for to, source in zip(holes, movers):
                (tp, ta), (sp, sa) = slots[to], slots[source]
                keys[tp, ta, g], values[tp, ta, g] = keys[sp, sa, g], values[sp, sa, g]
                weights[tp, g, ta], positions[tp, g, ta] = weights[sp, g, sa], positions[sp, g, sa]
            for j in range(budget, n):
                page, at = slots[j]
                weights[page, g, at], positions[page, g, at] = 0.0, -1
    return keys, values, weights, positions, torch.tensor(new, dtype=torch.int32)


def process_logits(logits, dtype=np.float64, *, history=None, history_lengths=None, prompt_lengths=None, repetition=None, presence=None,
                   frequency=None, bias_ids=None, bias_values=None, allowed=None):
    """(out, tokens): in ``dtype`` float64 the definition, in float32 its steps
    with each rounded."""
    x = cpu(logits).float().numpy().astype(dtype)
    rows, vocab = x.shape
    at = lambda t, r, default: dtype(default if t is None else float(cpu(t)[r]))  # noqa: E731
    with np.errstate(all="ignore"):
        for r in range(rows):
            if history is not None:
                n = max(0, min(int(cpu(history_lengths)[r]), history.shape[1]))
                prompt = max(0, int(cpu(prompt_lengths)[r])) if prompt_lengths is not None else 0
                ids = cpu(history)[r, :n].numpy()
                fits = (ids >= 0) & (ids < vocab)
                seen = np.unique(ids[fits])
                rep = at(repetition, r, 1.0)
                x[r, seen] = np.where(x[r, seen] > 0, x[r, seen] / rep, x[r, seen] * rep)
                made, count = np.unique(ids[prompt:][fits[prompt:]], return_counts=True)
                x[r, made] = x[r, made] - at(frequency, r, 0.0) * count.astype(dtype) - at(presence, r, 0.0)
            if bias_ids is not None:
                last = {int(i): b for i, b in zip(cpu(bias_ids)[r], cpu(bias_values)[r].numpy())}
                for i, b in last.items():
                    if 0 <= i < vocab:
                        x[r, i] = x[r, i] + dtype(b)
            if allowed is not None:
                words = cpu(allowed)[r].numpy().view(np.uint32)
                bits = (words[:, None] >> np.arange(32, dtype=np.uint32) & 1).reshape(-1)[:vocab]
                x[r, bits == 0] = -np.inf
        tokens = [int(np.argmax(row)) if not np.isnan(row).any() and np.isfinite(row.max()) else -1 for row in x]
    return x, np.array(tokens, dtype=np.int64)
