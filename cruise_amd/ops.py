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
operators has a gradient: a tensor that requires one, input or output, is refused
while gradients are enabled, one with a forward-mode tangent always.
"""
from __future__ import annotations

import struct

import torch
from torch.autograd import forward_ad

from . import _lib

# The records of include/resident_epoch.h, and where the workspace's address and
# size lie in those that name one.
_CACHE = "4Q10q6i"
KV_WRITE = struct.Struct("<" + _CACHE + "9Q8q2ifi")
KV_ATTENTION = struct.Struct("<" + _CACHE + "5Q6q4ifi")
KV_EVICT = struct.Struct("<" + _CACHE + "5Q2q6i")
LOGITS = struct.Struct("<13Q7q6i")
_WORKSPACE = struct.Struct("<Qq")
_UNFIT = (struct.error, OverflowError)  # a number that its field cannot hold
_ATTENTION_AT = _EVICT_AT = struct.calcsize("<" + _CACHE + "4Q")
_LOGITS_AT = struct.calcsize("<12Q")

_BYTES = {torch.bfloat16: 2, torch.float32: 4}
_BF16, _F32, _I32, _I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64
_MAX_I32 = (1 << 31) - 1
_MOST_SLOTS = 1 << 30  # of a row

# A step of a few tokens takes a few microseconds on the GPU, so what a call
# costs on the host is what such a step costs: one comparison per property and
# tensor, names and messages only for a call that is refused, and the stream's
# handle without a Python object around it.
_raw_stream = torch._C._cuda_getCurrentRawStream


def _check(t, name: str, dtype, shape: tuple, gpu: int) -> None:
    """A tensor of this type and shape on GPU ``gpu``, its last dimension contiguous."""
    try:
        if t.dtype is dtype and t.get_device() == gpu and t.shape == shape and (t.is_contiguous() or t.stride(-1) == 1 or shape[-1] <= 1):
            return
    except AttributeError:
        pass
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.get_device() != gpu:
        raise ValueError(f"{name} must be a {dtype} tensor on cuda:{gpu}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, not {tuple(shape)}")
    raise ValueError(f"the last dimension of {name} must be contiguous")


def _address(t, name: str, dtype, rows: int, gpu: int) -> int:
    """The address of a vector of one value for each row; 0 for None."""
    if t is None:
        return 0
    _check(t, name, dtype, (rows,), gpu)
    return t.data_ptr()


def _gpu_of(t, name: str, dims: int) -> int:
    """The GPU of the tensor that says where a call runs."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a tensor on a GPU")
    if t.dtype not in _BYTES or t.dim() != dims:
        raise ValueError(f"{name} must be bfloat16 or float32, with {dims} dimensions")
    return t.get_device()


def _shape(t, name: str, dims: str, count: int):
    """The shape of a tensor whose sizes a call goes by."""
    if not isinstance(t, torch.Tensor) or t.dim() != count:
        raise ValueError(f"{name} must have the dimensions {dims}")
    return t.shape


def _no_gradients(names: str, *tensors) -> None:
    """Refuses tensors (None among them is none) that ask for a gradient, of either mode."""
    for i, t in enumerate(tensors):
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            break
    else:
        if forward_ad._current_level < 0:
            return
        for i, t in enumerate(tensors):
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                break
        else:
            return
    raise ValueError(f"{names.split()[i]} asks for a gradient, and the serving operators have none")


def _cache(keys, values, weights, positions, gpu: int) -> tuple:
    """The cache record's values, after its checks."""
    dtype, shape = keys.dtype, keys.shape
    pages, block, kv_heads, head_dim = shape
    k0, k1, k2, k3 = keys.stride()
    if k3 != 1:
        raise ValueError("the last dimension of key_cache must be contiguous")
    _check(values, "value_cache", dtype, shape, gpu)
    if head_dim not in (64, 128, 256):
        raise ValueError(f"head_dim is {head_dim}, not 64, 128 or 256")
    if not 0 < pages * block <= _MAX_I32 or not kv_heads:
        raise ValueError("a cache has at least one slot and fewer than 2^31")
    w = w0 = w1 = p = p0 = p1 = 0
    if weights is not None:
        _check(weights, "weight_cache", _F32, (pages, kv_heads, block), gpu)
        w, (w0, w1, _) = weights.data_ptr(), weights.stride()
    if positions is not None:
        _check(positions, "position_cache", _I32, (pages, kv_heads, block), gpu)
        p, (p0, p1, _) = positions.data_ptr(), positions.stride()
    v0, v1, v2, _ = values.stride()
    return (keys.data_ptr(), values.data_ptr(), w, p, k0, k1, k2, v0, v1, v2, w0, w1, p0, p1, pages, block, kv_heads, head_dim, _BYTES[dtype],
            gpu)


def _bound(block_table, block: int, max_length) -> int:
    """The most slots that a row can have."""
    bound = min(_MOST_SLOTS, block_table.shape[1] * block)
    if max_length is None:
        return bound
    if max_length < 0:
        raise ValueError("max_length is negative")
    return min(bound, max_length)


def _unfit(name: str, why: Exception) -> ValueError:
    return ValueError(f"{name}: a number of the wrong type or out of range ({why})")


def _done(code: int, name: str) -> None:
    if code == -1:
        raise ValueError(f"{name} refused its arguments: rows of elements start at multiples of 16 bytes, and the limits and "
                         "overlaps of include/resident_epoch.h hold")
    if code != 0:
        raise RuntimeError(f"{name} failed: {code}")


def _with_workspace(size: int, name: str, record: bytes, at: int, gpu: int) -> tuple:
    """The record with a workspace of ``size`` bytes, and what keeps it alive
    until the call is queued.  It comes from torch's allocator, so that two
    calls at once, or two captured graphs, never share one."""
    if size < 0:
        _done(-1, name)
    if size == 0:
        return record, None
    workspace = torch.empty(size, dtype=torch.uint8, device=gpu)
    return record[:at] + _WORKSPACE.pack(workspace.data_ptr(), size) + record[at + 16 :], workspace


def kv_write(q, k, v, positions, slots, key_cache, value_cache, inv_freq, *, q_norm=None, k_norm=None, eps: float = 1e-6,
             weight_cache=None, position_cache=None, out=None) -> torch.Tensor:
    """New tokens into the cache (``resident_kv_write``); returns the rotated queries.

    q ``[tokens, heads, head_dim]``, k and v ``[tokens, kv_heads, head_dim]`` of
    the caches' type (views of one projection's output will do), positions
    int64 ``[tokens]`` (below 2^31), slots int32 ``[tokens]`` (a slot outside the
    pool: the token is not stored), inv_freq fp32 ``[head_dim / 2]``.  q_norm and
    k_norm ``[head_dim]`` scale the heads after their RMS norm; without them
    heads are rotated as they are.  ``out`` may be ``q``, or lies apart from what the
    call uses (other parts of one projection are apart)."""
    gpu = _gpu_of(key_cache, "key_cache", 4)
    cache = _cache(key_cache, value_cache, weight_cache, position_cache, gpu)
    dtype, (_, _, kv_heads, d) = key_cache.dtype, key_cache.shape
    tokens, heads, _ = _shape(q, "q", "[tokens, heads, head_dim]", 3)
    if not heads:
        raise ValueError("q has no heads")
    _check(q, "q", dtype, (tokens, heads, d), gpu)
    _check(k, "k", dtype, (tokens, kv_heads, d), gpu)
    _check(v, "v", dtype, (tokens, kv_heads, d), gpu)
    _check(positions, "positions", _I64, (tokens,), gpu)
    _check(slots, "slots", _I32, (tokens,), gpu)
    _check(inv_freq, "inv_freq", _F32, (d // 2,), gpu)
    qn, kn = _address(q_norm, "q_norm", dtype, d, gpu), _address(k_norm, "k_norm", dtype, d, gpu)
    if out is not None:
        _check(out, "out", dtype, (tokens, heads, d), gpu)
    _no_gradients("q k v key_cache value_cache weight_cache q_norm k_norm inv_freq out", q, k, v, key_cache, value_cache, weight_cache, q_norm,
                  k_norm, inv_freq, out)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if tokens:
        (q0, q1, _), (k0, k1, _), (v0, v1, _), (o0, o1, _) = q.stride(), k.stride(), v.stride(), out.stride()
        try:
            record = KV_WRITE.pack(*cache, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), qn, kn, inv_freq.data_ptr(),
                                   positions.data_ptr(), slots.data_ptr(), q0, q1, k0, k1, v0, v1, o0, o1, tokens, heads, eps, 0)
        except _UNFIT as why:
            raise _unfit("resident_kv_write", why) from None
        code = _lib.load().resident_kv_write(record, _raw_stream(gpu))
        if code:
            _done(code, "resident_kv_write")
    return out


def kv_attention(q, key_cache, value_cache, block_table, lengths, *, scale: float | None = None, weight_cache=None,
                 max_length: int | None = None, out=None) -> torch.Tensor:
    """One new token of every row over the row's slots (``resident_kv_attention``).

    q ``[rows, heads, head_dim]`` of the caches' type, heads a multiple of the
    cache's.  ``scale`` defaults to head_dim^-0.5.  ``max_length`` is a bound of
    the lengths that the caller knows (they are cut to it; the default is what
    the table can hold): launch and workspace are sized by it, so a close one is
    faster and smaller (the scores of every query head are kept for the weights).
    Where ``weight_cache`` is given, every slot's weight grows by the attention
    that its KV head's queries give it (no page may then be named twice).  ``out`` may be ``q``, or lies apart from what the call uses."""
    gpu = _gpu_of(key_cache, "key_cache", 4)
    cache = _cache(key_cache, value_cache, weight_cache, None, gpu)
    dtype, (_, block, kv_heads, d) = key_cache.dtype, key_cache.shape
    rows, heads, _ = _shape(q, "q", "[rows, heads, head_dim]", 3)
    if not heads or heads % kv_heads:
        raise ValueError("the query heads must be a multiple of the cache's KV heads")
    _check(q, "q", dtype, (rows, heads, d), gpu)
    _, width = _shape(block_table, "block_table", "[rows, width]", 2)
    _check(block_table, "block_table", _I32, (rows, width), gpu)
    _check(lengths, "lengths", _I32, (rows,), gpu)
    bound = _bound(block_table, block, max_length)
    if out is not None:
        _check(out, "out", dtype, (rows, heads, d), gpu)
    _no_gradients("q key_cache value_cache weight_cache out", q, key_cache, value_cache, weight_cache, out)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if rows:
        (q0, q1, _), (o0, o1, _) = q.stride(), out.stride()
        try:
            record = KV_ATTENTION.pack(*cache, q.data_ptr(), out.data_ptr(), block_table.data_ptr(), lengths.data_ptr(), 0, 0, q0, q1, o0, o1,
                                       block_table.stride(0), rows, heads, width, bound, d**-0.5 if scale is None else scale, 0)
        except _UNFIT as why:
            raise _unfit("resident_kv_attention", why) from None
        lib = _lib.load()
        record, _keep = _with_workspace(lib.resident_kv_attention_workspace(record), "resident_kv_attention", record, _ATTENTION_AT, gpu)
        code = lib.resident_kv_attention(record, _raw_stream(gpu))
        if code:
            _done(code, "resident_kv_attention")
    return out


def kv_evict(key_cache, value_cache, block_table, lengths, next_positions, weight_cache, position_cache, *, budget: int, recent: int,
             sinks: int = 0, max_length: int | None = None, out_lengths=None) -> torch.Tensor:
    """Every KV head of a row keeps ``budget`` slots (``resident_kv_evict``);
    returns the new lengths, min(length, budget), int32 ``[rows]``, which are the
    next step's: every layer of one step takes the lengths that it began with.

    Kept are the tokens of the last ``recent`` positions before
    ``next_positions`` (int64 ``[rows]``) and of the first ``sinks``, then the
    slots of greatest weight.  The order of slots is not kept: position_cache
    says which token a slot holds.  Of more protected slots than the budget the lowest
    stay.  No page may be named twice.  ``max_length`` as
    in ``kv_attention``."""
    gpu = _gpu_of(key_cache, "key_cache", 4)
    if weight_cache is None or position_cache is None:
        raise ValueError("eviction needs weight_cache and position_cache")
    cache = _cache(key_cache, value_cache, weight_cache, position_cache, gpu)
    rows, width = _shape(block_table, "block_table", "[rows, width]", 2)
    _check(block_table, "block_table", _I32, (rows, width), gpu)
    _check(lengths, "lengths", _I32, (rows,), gpu)
    _check(next_positions, "next_positions", _I64, (rows,), gpu)
    if not 0 < budget <= _MAX_I32 or recent < 0 or sinks < 0 or recent + sinks > budget:
        raise ValueError("budget must be positive, and recent + sinks at most the budget")
    _no_gradients("key_cache value_cache weight_cache", key_cache, value_cache, weight_cache)
    bound = _bound(block_table, key_cache.shape[1], max_length)
    if out_lengths is None:
        out_lengths = torch.empty(rows, dtype=_I32, device=gpu)
    else:
        _check(out_lengths, "out_lengths", _I32, (rows,), gpu)
    if rows:
        try:
            record = KV_EVICT.pack(*cache, block_table.data_ptr(), lengths.data_ptr(), next_positions.data_ptr(), out_lengths.data_ptr(), 0, 0,
                                   block_table.stride(0), rows, width, bound, budget, recent, sinks)
        except _UNFIT as why:
            raise _unfit("resident_kv_evict", why) from None
        lib = _lib.load()
        record, _keep = _with_workspace(lib.resident_kv_evict_workspace(record), "resident_kv_evict", record, _EVICT_AT, gpu)
        code = lib.resident_kv_evict(record, _raw_stream(gpu))
        if code:
            _done(code, "resident_kv_evict")
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
    ``[rows, biases]`` (of an id that is named twice the last value counts); allowed int32 ``[rows, ceil(vocab / 32)]``, a bit for each
    id, lowest first.  ``out`` may be ``logits``."""
    gpu = _gpu_of(logits, "logits", 2)
    rows, vocab = logits.shape
    l0, l1 = logits.stride()
    if not 0 < vocab <= _MAX_I32 or (l1 != 1 and vocab > 1):
        raise ValueError("logits must have a vocabulary, and it must be contiguous")
    h = hs = width = b = bv = bs = bvs = biases = al = als = 0
    if history is not None:
        if history_lengths is None:
            raise ValueError("history needs history_lengths")
        _, width = _shape(history, "history", "[rows, width]", 2)
        _check(history, "history", _I64, (rows, width), gpu)
        if width:
            h, hs = history.data_ptr(), history.stride(0)
    hl = _address(history_lengths, "history_lengths", _I32, rows, gpu)
    pl = _address(prompt_lengths, "prompt_lengths", _I32, rows, gpu)
    if bias_ids is not None:
        _, biases = _shape(bias_ids, "bias_ids", "[rows, biases]", 2)
        _check(bias_ids, "bias_ids", _I64, (rows, biases), gpu)
        _check(bias_values, "bias_values", _F32, (rows, biases), gpu)
        if biases:
            b, bs, bv, bvs = bias_ids.data_ptr(), bias_ids.stride(0), bias_values.data_ptr(), bias_values.stride(0)
    if allowed is not None:
        _check(allowed, "allowed", _I32, (rows, (vocab + 31) // 32), gpu)
        al, als = allowed.data_ptr(), allowed.stride(0)
    rep = _address(repetition, "repetition", _F32, rows, gpu)
    pres = _address(presence, "presence", _F32, rows, gpu)
    freq = _address(frequency, "frequency", _F32, rows, gpu)
    if out is not None:
        _check(out, "out", _F32, (rows, vocab), gpu)
    _no_gradients("logits repetition presence frequency bias_values out", logits, repetition, presence, frequency,
                  None if bias_ids is None else bias_values, out)
    if out is None:
        out = torch.empty_like(logits, dtype=_F32, memory_format=torch.contiguous_format)
    if tokens is None:
        tokens = torch.empty(rows, dtype=_I64, device=gpu)
    else:
        _check(tokens, "tokens", _I64, (rows,), gpu)
    if rows:
        try:
            record = LOGITS.pack(logits.data_ptr(), out.data_ptr(), tokens.data_ptr(), h, hl, pl, rep, pres, freq, b, bv, al, 0, 0, l0,
                                 out.stride(0), hs, bs, bvs, als, rows, vocab, width, biases, _BYTES[logits.dtype], gpu)
        except _UNFIT as why:
            raise _unfit("resident_logits_process", why) from None
        lib = _lib.load()
        record, _keep = _with_workspace(lib.resident_logits_process_workspace(record), "resident_logits_process", record, _LOGITS_AT, gpu)
        code = lib.resident_logits_process(record, _raw_stream(gpu))
        if code:
            _done(code, "resident_logits_process")
    return out, tokens
