"""Serving operators on torch tensors: a decode loop outside the resident epoch.

Over one layer's paged cache at a time (``key_cache[layer]`` of the decoder-step ABI
is one):

* ``kv_write``             -- norm of each query and key head, rotation by the token's
  position, keys and values to their slots;
* ``kv_attention``         -- one new token of every row over the row's slots, adding
  the attention weight of each slot to the cache's weights if it has any;
* ``kv_prefix_attention``  -- the same behind a prefix that all rows share, computed
  once for all of them;
* ``kv_evict``             -- every KV head keeps its ``budget`` slots of greatest weight;

and around it:

* ``block_norms``          -- the norm after a block, its gate and residual scale, the
  residual sum and the norm before the next block;
* ``quantize_rows``, ``int8_linear`` -- projections in 8-bit integers with a scale for
  each token and output channel;
* ``process_logits``       -- penalties, biases, a grammar mask and the greedy token.

They need no engine, queue their work on the current stream of the tensors'
device, do not wait for it, and may be captured into a graph.  What each
computes, and what it does with bad pages, empty rows and ties, is said at its
record in ``include/resident_epoch.h``.  Arguments that do not fit raise
``ValueError`` before anything is queued, a failed launch ``RuntimeError``.

Shapes: caches ``[pages, block, kv_heads, head_dim]`` (bf16 or fp32, head_dim
64, 128 or 256), weights and positions ``[pages, kv_heads, block]`` (fp32,
int32), block tables int32 ``[rows, width]``, lengths int32 ``[rows]``.  Views
with other strides are taken as they are, as long as the last dimension is
contiguous and rows of elements of the cache operators and of 8-bit matrices start at
multiples of 16 bytes (rows of ``block_norms``, ``quantize_rows`` and bf16 or fp32 rows
of ``int8_linear`` may start at any element).  None of the operators has a gradient: a
tensor that requires one, input or output, is refused while gradients are enabled, one
with a forward-mode tangent always.
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
KV_PREFIX_ATTENTION = struct.Struct(KV_ATTENTION.format + "2Q2i")
KV_EVICT = struct.Struct("<" + _CACHE + "5Q2q6i")
LOGITS = struct.Struct("<13Q7q6i")
BLOCK_NORMS = struct.Struct("<8Q6q4i2f")
QUANTIZE_ROWS = struct.Struct("<3Q2q4i")
INT8_LINEAR = struct.Struct("<7Q4q6i")
_WORKSPACE = struct.Struct("<Qq")
_UNFIT = (struct.error, OverflowError)  # a number that its field cannot hold
_ATTENTION_AT = _EVICT_AT = struct.calcsize("<" + _CACHE + "4Q")
_LOGITS_AT = struct.calcsize("<12Q")
_LINEAR_AT = struct.calcsize("<6Q")

_BYTES = {torch.bfloat16: 2, torch.float32: 4}
_BF16, _F32, _I8, _I32, _I64 = torch.bfloat16, torch.float32, torch.int8, torch.int32, torch.int64
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


def _bound(width: int, block: int, max_length, name: str = "max_length") -> int:
    """The most slots that a row of a table of this width can have."""
    bound = min(_MOST_SLOTS, width * block)
    if max_length is None:
        return bound
    if max_length < 0:
        raise ValueError(f"{name} is negative")
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
    bound = _bound(width, block, max_length)
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


def kv_prefix_attention(q, key_cache, value_cache, prefix_table, prefix_length, block_table, lengths, *, scale: float | None = None,
                        weight_cache=None, max_prefix: int | None = None, max_length: int | None = None, out=None) -> torch.Tensor:
    """One new token of every row over a prefix that all rows share, computed once
    for all, and over the row's own slots (``resident_kv_prefix_attention``).

    prefix_table int32 ``[width]`` names the prefix's pages and prefix_length int32
    ``[1]`` its slots; ``block_table`` and ``lengths`` are the rows' own, what came after
    the prefix.  Everything else is as in ``kv_attention``, ``max_prefix`` for the
    prefix what ``max_length`` is for the rows.  Where ``weight_cache`` is given, the
    weights of the rows' own slots grow, so that ``kv_evict`` can be called on them; the
    prefix's stay as they are."""
    gpu = _gpu_of(key_cache, "key_cache", 4)
    cache = _cache(key_cache, value_cache, weight_cache, None, gpu)
    dtype, (_, block, kv_heads, d) = key_cache.dtype, key_cache.shape
    rows, heads, _ = _shape(q, "q", "[rows, heads, head_dim]", 3)
    if not heads or heads % kv_heads:
        raise ValueError("the query heads must be a multiple of the cache's KV heads")
    _check(q, "q", dtype, (rows, heads, d), gpu)
    (prefix_width,) = _shape(prefix_table, "prefix_table", "[width]", 1)
    _check(prefix_table, "prefix_table", _I32, (prefix_width,), gpu)
    _check(prefix_length, "prefix_length", _I32, (1,), gpu)
    _, width = _shape(block_table, "block_table", "[rows, width]", 2)
    _check(block_table, "block_table", _I32, (rows, width), gpu)
    _check(lengths, "lengths", _I32, (rows,), gpu)
    prefix_bound, bound = _bound(prefix_width, block, max_prefix, "max_prefix"), _bound(width, block, max_length)
    if out is not None:
        _check(out, "out", dtype, (rows, heads, d), gpu)
    _no_gradients("q key_cache value_cache weight_cache out", q, key_cache, value_cache, weight_cache, out)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if rows:
        (q0, q1, _), (o0, o1, _) = q.stride(), out.stride()
        try:
            record = KV_PREFIX_ATTENTION.pack(*cache, q.data_ptr(), out.data_ptr(), block_table.data_ptr(), lengths.data_ptr(), 0, 0, q0, q1, o0,
                                              o1, block_table.stride(0), rows, heads, width, bound, d**-0.5 if scale is None else scale, 0,
                                              prefix_table.data_ptr(), prefix_length.data_ptr(), prefix_width, prefix_bound)
        except _UNFIT as why:
            raise _unfit("resident_kv_prefix_attention", why) from None
        lib = _lib.load()
        record, _keep = _with_workspace(lib.resident_kv_prefix_attention_workspace(record), "resident_kv_prefix_attention", record, _ATTENTION_AT,
                                        gpu)
        code = lib.resident_kv_prefix_attention(record, _raw_stream(gpu))
        if code:
            _done(code, "resident_kv_prefix_attention")
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
    bound = _bound(width, key_cache.shape[1], max_length)
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


def block_norms(x, residual, *, pre_norm, post_norm=None, gate=None, scale: float = 1.0, eps: float = 1e-6, quantize: bool = False,
                residual_out=None, out=None, out_scales=None):
    """The norm after a block, its gate and residual scale, the residual sum and the
    norm before the next block (``resident_block_norms``); returns the new residual
    and the normed rows, with ``quantize`` the latter as int8 and their scales, as
    ``quantize_rows`` would give them.

    x and residual ``[tokens, hidden]`` bf16 or fp32, hidden up to 32,768; post_norm
    and pre_norm ``[hidden]``; gate ``[hidden]``, ``[tokens, 1]`` or ``[tokens,
    hidden]``.  Without x (None: before the first block) the residual is returned as it
    is, and ``out`` lies apart from it.  Otherwise ``residual_out`` and ``out`` may be
    ``x``, ``residual`` or a gate of a value for each token and channel, not both the same."""
    gpu = _gpu_of(residual, "residual", 2)
    dtype, shape = residual.dtype, residual.shape
    tokens, hidden = shape
    if not hidden:
        raise ValueError("residual has no channels")
    _check(residual, "residual", dtype, shape, gpu)
    _check(pre_norm, "pre_norm", dtype, (hidden,), gpu)
    post = _address(post_norm, "post_norm", dtype, hidden, gpu)
    xp = xs = gp = g0 = g1 = sp = 0
    if x is not None:
        _check(x, "x", dtype, shape, gpu)
        xp, xs = x.data_ptr(), x.stride(0)
    elif post_norm is not None or gate is not None or residual_out is not None:
        raise ValueError("post_norm, gate and residual_out need x")
    if gate is not None:
        if isinstance(gate, torch.Tensor) and gate.dim() == 1:
            _check(gate, "gate", dtype, (hidden,), gpu)
            g1 = 1
        elif isinstance(gate, torch.Tensor) and gate.shape == (tokens, 1):
            _check(gate, "gate", dtype, (tokens, 1), gpu)
            g0 = gate.stride(0)
        else:
            _check(gate, "gate", dtype, shape, gpu)
            g0, g1 = gate.stride(0), 1
        gp = gate.data_ptr()
    if residual_out is not None:
        _check(residual_out, "residual_out", dtype, shape, gpu)
    if out is not None:
        _check(out, "out", _I8 if quantize else dtype, shape, gpu)
    if out_scales is not None:
        if not quantize:
            raise ValueError("out_scales needs quantize")
        _check(out_scales, "out_scales", _F32, (tokens,), gpu)
    _no_gradients("x residual pre_norm post_norm gate residual_out out out_scales", x, residual, pre_norm, post_norm, gate, residual_out, out,
                  out_scales)
    if x is None:
        residual_out = residual
    elif residual_out is None:
        residual_out = torch.empty_like(residual, memory_format=torch.contiguous_format)
    if out is None:
        out = torch.empty(shape, dtype=_I8 if quantize else dtype, device=gpu)
    if quantize and out_scales is None:
        out_scales = torch.empty(tokens, dtype=_F32, device=gpu)
    if x is not None:
        sp = residual_out.data_ptr()
    if tokens:
        try:
            record = BLOCK_NORMS.pack(xp, residual.data_ptr(), post, gp, pre_norm.data_ptr(), sp, out.data_ptr(),
                                      out_scales.data_ptr() if quantize else 0, xs, residual.stride(0), residual_out.stride(0), out.stride(0), g0,
                                      g1, tokens, hidden, _BYTES[dtype], gpu, eps, scale)
        except _UNFIT as why:
            raise _unfit("resident_block_norms", why) from None
        code = _lib.load().resident_block_norms(record, _raw_stream(gpu))
        if code:
            _done(code, "resident_block_norms")
    return (residual_out, out, out_scales) if quantize else (residual_out, out)


def quantize_rows(x, *, out=None, scales=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows to 8-bit integers (``resident_quantize_rows``); returns them, int8, and
    each row's scale, fp32 ``[rows]``: the greatest magnitude is 127 of it.

    x bf16 or fp32 ``[rows, columns]``.  The same call lays out weights ``[outer,
    inner]`` for ``int8_linear`` with a scale for each output channel."""
    gpu = _gpu_of(x, "x", 2)
    rows, columns = x.shape
    if not columns:
        raise ValueError("x has no columns")
    _check(x, "x", x.dtype, x.shape, gpu)
    if out is not None:
        _check(out, "out", _I8, x.shape, gpu)
    if scales is not None:
        _check(scales, "scales", _F32, (rows,), gpu)
    _no_gradients("x scales", x, scales)
    if out is None:
        out = torch.empty(x.shape, dtype=_I8, device=gpu)
    if scales is None:
        scales = torch.empty(rows, dtype=_F32, device=gpu)
    if rows:
        try:
            record = QUANTIZE_ROWS.pack(x.data_ptr(), out.data_ptr(), scales.data_ptr(), x.stride(0), out.stride(0), rows, columns,
                                        _BYTES[x.dtype], gpu)
        except _UNFIT as why:
            raise _unfit("resident_quantize_rows", why) from None
        code = _lib.load().resident_quantize_rows(record, _raw_stream(gpu))
        if code:
            _done(code, "resident_quantize_rows")
    return out, scales


def int8_linear(x, weight, weight_scale, *, x_scale=None, bias=None, dtype=None, out=None) -> torch.Tensor:
    """The product of rows with 8-bit weights (``resident_int8_linear``), ``[tokens,
    outer]``.

    weight int8 ``[outer, inner]`` with weight_scale fp32 ``[outer]`` (``quantize_rows``
    gives both); x bf16 or fp32 ``[tokens, inner]``, which the call brings to 8 bits, or
    int8 with x_scale fp32 ``[tokens]`` (several projections of the same rows share
    one ``quantize_rows``, or ``block_norms`` with ``quantize``).  The result is of
    ``dtype`` (bf16 or fp32; x's, bf16 where that is int8), and so is the bias
    ``[outer]``.  inner is a multiple of 16."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError("x must be a tensor on a GPU")
    given = x.dtype
    if (given not in _BYTES and given is not _I8) or x.dim() != 2:
        raise ValueError("x must be bfloat16, float32 or int8, with 2 dimensions")
    gpu = x.get_device()
    if dtype is None:
        dtype = out.dtype if isinstance(out, torch.Tensor) else _BF16 if given is _I8 else given
    if dtype not in _BYTES:
        raise ValueError("the result must be bfloat16 or float32")
    tokens, inner = x.shape
    outer, _ = _shape(weight, "weight", "[outer, inner]", 2)
    if not outer or not inner:
        raise ValueError("weight has no channels")
    _check(x, "x", given, (tokens, inner), gpu)
    _check(weight, "weight", _I8, (outer, inner), gpu)
    _check(weight_scale, "weight_scale", _F32, (outer,), gpu)
    if (x_scale is None) == (given is _I8):
        raise ValueError("x_scale belongs to an x in 8 bits, and to no other")
    xs, b = _address(x_scale, "x_scale", _F32, tokens, gpu), _address(bias, "bias", dtype, outer, gpu)
    if out is not None:
        _check(out, "out", dtype, (tokens, outer), gpu)
    _no_gradients("x weight_scale x_scale bias out", x, weight_scale, x_scale, bias, out)
    if out is None:
        out = torch.empty(tokens, outer, dtype=dtype, device=gpu)
    if tokens:
        try:
            record = INT8_LINEAR.pack(x.data_ptr(), xs, weight.data_ptr(), weight_scale.data_ptr(), b, out.data_ptr(), 0, 0, x.stride(0),
                                      weight.stride(0), out.stride(0), tokens, inner, outer, 1 if given is _I8 else _BYTES[given], _BYTES[dtype],
                                      gpu)
        except _UNFIT as why:
            raise _unfit("resident_int8_linear", why) from None
        lib = _lib.load()
        record, _keep = _with_workspace(lib.resident_int8_linear_workspace(record), "resident_int8_linear", record, _LINEAR_AT, gpu)
        code = lib.resident_int8_linear(record, _raw_stream(gpu))
        if code:
            _done(code, "resident_int8_linear")
    return out
