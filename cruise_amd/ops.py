"""Serving operators over a caller's paged cache, on torch tensors.

A decode loop outside the resident epoch, for one layer's cache at a time
(``key_cache[layer]`` of the decoder-step ABI is one):

* ``kv_write``        -- norm of each query and key head, rotation by the token's
  position, keys and values to their slots;
* ``kv_attention``    -- one new token of every row over the row's slots, adding
  the attention weight of each slot to the cache's weights if it has any;
* ``kv_evict``        -- every KV head keeps its ``budget`` slots of greatest weight;
* ``process_logits``  -- penalties, biases, a grammar mask and the greedy token.

They need no engine, queue their work on the current stream of the tensors'
device, do not wait for it, and may be captured into a graph.  What each
computes, and what it does with bad pages, empty rows and ties, is said at its
record in ``include/resident_epoch.h``.  Arguments that do not fit raise
``ValueError`` before anything is queued, a failed launch ``RuntimeError``.

Shapes: caches ``[pages, block, kv_heads, head_dim]`` (bf16 or fp32, head_dim
64, 128 or 256), weights and positions ``[pages, kv_heads, block]`` (fp32,
int32), block tables int32 ``[rows, width]``, lengths int32 ``[rows]``.  Views
with other strides are taken as they are, as long as the last dimension is
contiguous and rows of elements start at multiples of 16 bytes.  None of the
operators has a gradient.
"""
from __future__ import annotations

import struct

import torch

from . import _lib

# The records of include/resident_epoch.h.
_CACHE = "4Q10q6i"
KV_WRITE = struct.Struct("<" + _CACHE + "9Q8q2ifi")
KV_ATTENTION = struct.Struct("<" + _CACHE + "5Q6q4ifi")
KV_EVICT = struct.Struct("<" + _CACHE + "5Q2q6i")
LOGITS = struct.Struct("<13Q7q6i")

_BYTES = {torch.bfloat16: 2, torch.float32: 4}
_MAX_I32 = (1 << 31) - 1


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _check(t, name: str, dtype, shape, device) -> None:
    """A tensor of the given type and shape (None: any size) on ``device``,
    its last dimension contiguous."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be a {dtype} tensor on {device}")
    got = t.shape
    if len(got) != len(shape) or any(w is not None and w != g for w, g in zip(shape, got)):
        raise ValueError(f"{name} has shape {tuple(got)}, not {tuple('any' if w is None else w for w in shape)}")
    if got[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")


def _check_rows(t, name: str, dtype, rows: int, device) -> int:
    """The address of a contiguous vector of one value for each row; 0 for None."""
    if t is None:
        return 0
    _check(t, name, dtype, (rows,), device)
    return t.data_ptr()


def _gpu(t, name: str) -> torch.device:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a tensor on a GPU")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} asks for a gradient, and the serving operators have none")
    return t.device


def _cache(keys, values, weights, positions) -> tuple:
    """The cache record's values, after its checks."""
    device = _gpu(keys, "key_cache")
    dtype = keys.dtype
    _need(dtype in _BYTES, "key_cache must be bfloat16 or float32")
    _need(keys.dim() == 4, "key_cache must have the dimensions [pages, block, kv_heads, head_dim]")
    pages, block, kv_heads, head_dim = shape = keys.shape
    _check(keys, "key_cache", dtype, shape, device)
    _check(values, "value_cache", dtype, shape, device)
    _need(head_dim in (64, 128, 256), f"head_dim is {head_dim}, not 64, 128 or 256")
    _need(0 < pages * block <= _MAX_I32 and kv_heads > 0, "a cache has at least one slot and fewer than 2^31")
    ks, vs = keys.stride(), values.stride()
    w = p = 0
    wst = pst = (0, 0)
    if weights is not None:
        _check(weights, "weight_cache", torch.float32, (pages, kv_heads, block), device)
        w, wst = weights.data_ptr(), weights.stride()
    if positions is not None:
        _check(positions, "position_cache", torch.int32, (pages, kv_heads, block), device)
        p, pst = positions.data_ptr(), positions.stride()
    return (keys.data_ptr(), values.data_ptr(), w, p, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], wst[0], wst[1], pst[0], pst[1],
            pages, block, kv_heads, head_dim, _BYTES[dtype], device.index)


def _call(name: str, record: bytes, device: torch.device) -> None:
    code = getattr(_lib.load(), name)(record, torch.cuda.current_stream(device).cuda_stream)
    if code == -1:
        raise ValueError(f"{name} refused its arguments: rows of elements start at multiples of 16 bytes, and the limits and "
                         "overlaps of include/resident_epoch.h hold")
    if code != 0:
        raise RuntimeError(f"{name} failed: {code}")


def _workspace(name: str, record: bytes, device: torch.device):
    """A workspace for the call from torch's allocator (so two calls at once,
    or two captured graphs, never share one); None where none is needed."""
    size = getattr(_lib.load(), name)(record)
    if size < 0:
        raise ValueError(f"{name} refused the arguments: rows of elements start at multiples of 16 bytes, and the limits and "
                         "overlaps of include/resident_epoch.h hold")
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def kv_write(q, k, v, positions, slots, key_cache, value_cache, inv_freq, *, q_norm=None, k_norm=None, eps: float = 1e-6,
             weight_cache=None, position_cache=None, out=None) -> torch.Tensor:
    """New tokens into the cache (``resident_kv_write``); returns the rotated queries.

    q ``[tokens, heads, head_dim]``, k and v ``[tokens, kv_heads, head_dim]`` of
    the caches' type (views of one projection's output will do), positions
    int64 ``[tokens]`` (below 2^31), slots int32 ``[tokens]`` (a slot outside the
    pool: the token is not stored), inv_freq fp32 ``[head_dim / 2]``.  q_norm and
    k_norm ``[head_dim]`` scale the heads after their RMS norm; without them
    heads are rotated as they are.  ``out`` may be ``q``."""
    device = _gpu(key_cache, "key_cache")
    cache = _cache(key_cache, value_cache, weight_cache, position_cache)
    dtype, kv_heads, d = key_cache.dtype, key_cache.shape[2], key_cache.shape[3]
    _gpu(q, "q"), _gpu(k, "k"), _gpu(v, "v")
    _check(q, "q", dtype, (None, None, d), device)
    tokens, heads, _ = q.shape
    _need(heads > 0, "q has no heads")
    _check(k, "k", dtype, (tokens, kv_heads, d), device)
    _check(v, "v", dtype, (tokens, kv_heads, d), device)
    _check(positions, "positions", torch.int64, (tokens,), device)
    _check(slots, "slots", torch.int32, (tokens,), device)
    _check(inv_freq, "inv_freq", torch.float32, (d // 2,), device)
    norms = [0, 0]
    for i, (norm, name) in enumerate(((q_norm, "q_norm"), (k_norm, "k_norm"))):
        if norm is not None:
            _check(norm, name, dtype, (d,), device)
            norms[i] = norm.data_ptr()
    if out is None:
        out = torch.empty((tokens, heads, d), dtype=dtype, device=device)
    else:
        _check(out, "out", dtype, (tokens, heads, d), device)
    if tokens == 0:
        return out
    qs, ks, vs, os = q.stride(), k.stride(), v.stride(), out.stride()
    _call("resident_kv_write", KV_WRITE.pack(
        *cache, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), norms[0], norms[1], inv_freq.data_ptr(),
        positions.data_ptr(), slots.data_ptr(), qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os[0], os[1], tokens, heads, eps, 0), device)
    return out


def kv_attention(q, key_cache, value_cache, block_table, lengths, *, scale: float | None = None, weight_cache=None,
                 max_length: int | None = None, out=None) -> torch.Tensor:
    """One new token of every row over the row's slots (``resident_kv_attention``).

    q ``[rows, heads, head_dim]`` of the caches' type, heads a multiple of the
    cache's.  ``scale`` defaults to head_dim^-0.5.  ``max_length`` is a bound of
    the lengths that the caller knows (they are cut to it; the default is what the table can hold): the launch is
    sized by it, so a close one is faster.  Where ``weight_cache`` is given, every
    slot's weight grows by the attention that its KV head's queries give it.
    ``out`` may be ``q``."""
    device = _gpu(key_cache, "key_cache")
    cache = _cache(key_cache, value_cache, weight_cache, None)
    dtype, d = key_cache.dtype, key_cache.shape[3]
    _gpu(q, "q")
    _check(q, "q", dtype, (None, None, d), device)
    rows, heads, _ = q.shape
    _need(heads > 0 and heads % key_cache.shape[2] == 0, "the query heads must be a multiple of the cache's KV heads")
    _check(block_table, "block_table", torch.int32, (rows, None), device)
    _check(lengths, "lengths", torch.int32, (rows,), device)
    if out is None:
        out = torch.empty((rows, heads, d), dtype=dtype, device=device)
    else:
        _check(out, "out", dtype, (rows, heads, d), device)
    width = block_table.shape[1]
    bound = min(_MAX_I32, width * key_cache.shape[1])
    if max_length is not None:
        _need(max_length >= 0, "max_length is negative")
        bound = min(bound, max_length)
    if rows == 0:
        return out
    qs, os = q.stride(), out.stride()
    head = (*cache, q.data_ptr(), out.data_ptr(), block_table.data_ptr(), lengths.data_ptr())
    tail = (qs[0], qs[1], os[0], os[1], block_table.stride(0), rows, heads, width, bound, d**-0.5 if scale is None else scale, 0)
    workspace = _workspace("resident_kv_attention_workspace", KV_ATTENTION.pack(*head, 0, 0, *tail), device)
    at, size = (0, 0) if workspace is None else (workspace.data_ptr(), workspace.numel())
    _call("resident_kv_attention", KV_ATTENTION.pack(*head, at, size, *tail), device)
    return out


def kv_evict(key_cache, value_cache, block_table, lengths, next_positions, weight_cache, position_cache, *, budget: int, recent: int,
             sinks: int = 0, max_length: int | None = None, out_lengths=None) -> torch.Tensor:
    """Every KV head of a row keeps ``budget`` slots (``resident_kv_evict``);
    returns the new lengths, min(length, budget), int32 ``[rows]``.

    Kept are the tokens of the last ``recent`` positions before
    ``next_positions`` (int64 ``[rows]``) and of the first ``sinks``, then the
    slots of greatest weight.  The order of slots is not kept: position_cache
    says which token a slot holds.  Rows must not share pages."""
    device = _gpu(key_cache, "key_cache")
    _need(weight_cache is not None and position_cache is not None, "eviction needs weight_cache and position_cache")
    cache = _cache(key_cache, value_cache, weight_cache, position_cache)
    _need(isinstance(block_table, torch.Tensor) and block_table.dim() == 2, "block_table must have the dimensions [rows, width]")
    rows, width = block_table.shape
    _check(block_table, "block_table", torch.int32, (rows, width), device)
    _check(lengths, "lengths", torch.int32, (rows,), device)
    _check(next_positions, "next_positions", torch.int64, (rows,), device)
    _need(0 < budget <= _MAX_I32 and recent >= 0 and sinks >= 0 and recent + sinks <= budget,
          "budget must be positive, and recent + sinks at most the budget")
    if out_lengths is None:
        out_lengths = torch.empty(rows, dtype=torch.int32, device=device)
    else:
        _check(out_lengths, "out_lengths", torch.int32, (rows,), device)
    bound = min(_MAX_I32, width * key_cache.shape[1])
    if max_length is not None:
        _need(max_length >= 0, "max_length is negative")
        bound = min(bound, max_length)
    if rows == 0:
        return out_lengths
    head = (*cache, block_table.data_ptr(), lengths.data_ptr(), next_positions.data_ptr(), out_lengths.data_ptr())
    tail = (block_table.stride(0), rows, width, bound, budget, recent, sinks)
    workspace = _workspace("resident_kv_evict_workspace", KV_EVICT.pack(*head, 0, 0, *tail), device)
    at, size = (0, 0) if workspace is None else (workspace.data_ptr(), workspace.numel())
    _call("resident_kv_evict", KV_EVICT.pack(*head, at, size, *tail), device)
    return out_lengths


def process_logits(logits, *, history=None, history_lengths=None, prompt_lengths=None, repetition=None, presence=None, frequency=None,
                   bias_ids=None, bias_values=None, allowed=None, out=None, tokens=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Penalties, biases and a grammar mask (``resident_logits_process``);
    returns the processed logits, fp32 ``[rows, vocab]``, and each row's greedy
    token, int64 ``[rows]`` (-1: no finite choice).

    logits fp32 or bf16 ``[rows, vocab]``; history int64 ``[rows, width]`` with
    history_lengths int32 ``[rows]``, of which the first prompt_lengths int32
    ``[rows]`` are the prompt's (seen, but not generated); repetition, presence
    and frequency fp32 ``[rows]``; bias_ids int64 and bias_values fp32
    ``[rows, biases]``; allowed int32 ``[rows, ceil(vocab / 32)]``, a bit for each
    id, lowest first.  ``out`` may be ``logits``."""
    device = _gpu(logits, "logits")
    _need(logits.dtype in _BYTES, "logits must be bfloat16 or float32")
    _check(logits, "logits", logits.dtype, (None, None), device)
    rows, vocab = logits.shape
    _need(0 < vocab <= _MAX_I32, "logits have no vocabulary")
    h = hl = hs = hw = b = bv = bs = bvs = nb = al = als = 0
    pl = _check_rows(prompt_lengths, "prompt_lengths", torch.int32, rows, device)
    if history is not None:
        _check(history, "history", torch.int64, (rows, None), device)
        _need(history_lengths is not None, "history needs history_lengths")
        hw = history.shape[1]
        if hw:
            h, hs = history.data_ptr(), history.stride(0)
    hl = _check_rows(history_lengths, "history_lengths", torch.int32, rows, device)
    if bias_ids is not None:
        _check(bias_ids, "bias_ids", torch.int64, (rows, None), device)
        nb = bias_ids.shape[1]
        _need(bias_values is not None, "bias_ids need bias_values")
        _check(bias_values, "bias_values", torch.float32, (rows, nb), device)
        if nb:
            b, bs, bv, bvs = bias_ids.data_ptr(), bias_ids.stride(0), bias_values.data_ptr(), bias_values.stride(0)
    if allowed is not None:
        _check(allowed, "allowed", torch.int32, (rows, (vocab + 31) // 32), device)
        al, als = allowed.data_ptr(), allowed.stride(0)
    penalties = [_check_rows(t, n, torch.float32, rows, device)
                 for t, n in ((repetition, "repetition"), (presence, "presence"), (frequency, "frequency"))]
    if out is None:
        out = torch.empty((rows, vocab), dtype=torch.float32, device=device)
    else:
        _check(out, "out", torch.float32, (rows, vocab), device)
    if tokens is None:
        tokens = torch.empty(rows, dtype=torch.int64, device=device)
    else:
        _check(tokens, "tokens", torch.int64, (rows,), device)
    if rows == 0:
        return out, tokens
    head = (logits.data_ptr(), out.data_ptr(), tokens.data_ptr(), h, hl, pl, *penalties, b, bv, al)
    tail = (logits.stride(0), out.stride(0), hs, bs, bvs, als, rows, vocab, hw, nb, _BYTES[logits.dtype], device.index)
    workspace = _workspace("resident_logits_process_workspace", LOGITS.pack(*head, 0, 0, *tail), device)
    at, size = (0, 0) if workspace is None else (workspace.data_ptr(), workspace.numel())
    _call("resident_logits_process", LOGITS.pack(*head, at, size, *tail), device)
    return out, tokens
