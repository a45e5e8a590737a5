"""Attention behind a shared prefix, 8-bit products and the norms around a block
from their definitions, in 64 bits on the CPU: what the tests of cruise_amd.ops
compare with.  Every function returns a result and the tolerance that its
operator's rounding points give it."""
from __future__ import annotations

import numpy as np

from kv_ops_reference import HALF_STEP, cpu, slots_of, wide

STEP = 2.0**-24  # half an fp32 step: the largest relative error of one rounding
# What a probability beside a bf16 value is off by: it enters the product as two bf16 numbers.
TWO_PARTS = 2.0**-15


def prefix_attention(q, keys, values, prefix_table, prefix_length, table, lengths, scale=None, max_prefix=None, max_length=None):
    """(out, tolerance, gathered weights of the pool, their tolerance): the weights
    are what each slot is given, from 0."""
    dtype = q.dtype
    q, k, v = wide(q), wide(keys), wide(values)
    pages, block, kv_heads, d = k.shape
    rows, heads, _ = q.shape
    group = heads // kv_heads
    scale = d**-0.5 if scale is None else scale
    some = lambda width, bound: min(width * block, 1 << 30 if bound is None else bound)  # noqa: E731
    shared = slots_of(cpu(prefix_table), int(cpu(prefix_length)[0]), some(prefix_table.shape[0], max_prefix), pages, block)
    shared = [s for s in shared if s is not None]
    half = HALF_STEP[dtype]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    gathered, gathered_tol = np.zeros((pages, kv_heads, block)), np.zeros((pages, kv_heads, block))
    for r in range(rows):
        own = slots_of(cpu(table)[r], cpu(lengths)[r], some(table.shape[1], max_length), pages, block)
        slots = shared + [s for s in own if s is not None]
        if not slots:
            continue
        page, at = (np.array(x) for x in zip(*slots))
        for g in range(kv_heads):
            mine = slice(g * group, (g + 1) * group)
            kk, vv = k[page, at, g], v[page, at, g]
            s = scale * (q[r, mine] @ kk.T)
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            # fp32: the dot product of d terms and the scaling, of the slot and of the maximum; then exp, the sum of p
            # and the joining of parts.
            delta = 2 * abs(scale) * (np.abs(q[r, mine]) @ np.abs(kk).T).max(1, keepdims=True) * (d + 4) * STEP + (len(slots) + 32) * STEP
            size = p @ np.abs(vv)
            out[r, mine] = p @ vv
            tol[r, mine] = half * np.abs(out[r, mine]) + (delta + (TWO_PARTS if half > STEP else 0)) * size * (1 + half)
            n = len(shared)
            np.add.at(gathered, (page[n:], g, at[n:]), p[:, n:].sum(0))
            np.add.at(gathered_tol, (page[n:], g, at[n:]), (p[:, n:] * (delta + group * STEP)).sum(0))
    return out, tol, gathered, gathered_tol


def quantized(x):
    """The 8-bit rows and their scales, bit for bit: both quotients are fp32 ones."""
    x = cpu(x).float().numpy()
    with np.errstate(all="ignore"):
        scale = np.abs(x).max(1) / np.float32(127)
        q = np.rint(x / scale[:, None])
    bad = ~np.isfinite(x).all(1)
    q[(scale == 0) | bad] = 0
    scale[bad] = np.nan
    return np.clip(q, -127, 127).astype(np.int8), scale.astype(np.float32)


def product(x, x_scale, weight, weight_scale, bias, dtype):
    """(out, tolerance) of 8-bit rows times 8-bit weights: the sum is exact, then its
    conversion, the two products and the bias's sum are rounded to fp32, the result
    to its type."""
    total = np.asarray(x, dtype=np.float64) @ cpu(weight).double().numpy().T
    y = total * (np.asarray(x_scale, dtype=np.float64)[:, None] * wide(weight_scale))
    ref = y if bias is None else y + wide(bias)
    half = HALF_STEP[dtype]
    return ref, half * np.abs(ref) + (4 * STEP * np.abs(y) + STEP * np.abs(ref)) * (1 + half) + 2.0**-148


def norms(x, residual, pre_norm, post_norm=None, gate=None, scale=1.0, eps=1e-6):
    """(residual, tolerance, normed, tolerance before its rounding to the stored
    type): a lane sums up to 64 squares and up to 23 such sums are added, the root
    is off by a step, each product by half of one."""
    dtype = residual.dtype
    half, root = HALF_STEP[dtype], (87 / 2 + 4) * STEP
    r, off = wide(residual), 0.0
    n = r.shape[1]
    if x is not None:
        y = wide(x)
        if post_norm is not None:
            y = y / np.sqrt((y * y).sum(1, keepdims=True) / n + eps) * wide(post_norm)
        y = scale * y * (1 if gate is None else wide(gate))
        r = r + y
        off = (root + 6 * STEP) * np.abs(y) + STEP * np.abs(r)
    mean = (r * r).sum(1, keepdims=True) / n
    by = wide(pre_norm) / np.sqrt(mean + eps)
    out = r * by
    # What r is off by shows in the element itself and, through the mean, in all of the row.
    drift = np.sqrt(((off + np.zeros_like(r)) ** 2).sum(1, keepdims=True) / n / np.maximum(mean + eps, 1e-300))
    loose = np.abs(by) * off + np.abs(out) * (root + 3 * STEP + drift)
    return r, half * np.abs(r) + off * (1 + half), out, loose * (1 + half)
