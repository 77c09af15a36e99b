"""Attention over the paged pool: what a model computes with the keys and
values that the pool holds, without assembling them.

The reference's cache gathers a sequence's whole K and V per layer and leaves
the attention to the model (agentkv/hf_cache.py:129-153).  Here a decode step
works on the pool ``[blocks, layers, 2, kv_heads, block_size, head_dim]``
itself, for a batch of sequences at once:

* ``kv_append``        the new tokens' keys (rotated by position on the way, and
                       the queries with them) and values into their blocks;
* ``paged_attention``  the attention of one new token per sequence, over all its
                       positions, the last ``window`` of them, or selected blocks;
* ``select_blocks``    the blocks that matter most to the new token, ranked by
                       their ``key_bounds`` (kept up to date by ``kv_append``).

A batch is ``tables`` (int32 ``[rows, width]``: row s's token t lies in block
``tables[s, t // block_size]``) and ``lengths`` (int32 ``[rows]``: the tokens that
row s holds, the new ones among them; 0 for a padding row).  Entries behind a
row's last block are never read.  ``DecodeBatch`` keeps both for a set of
agents.

Every call is enqueued on the pool's device's current stream and does not
wait; its work space comes from PyTorch's allocator for that stream, so calls
on several streams and captured calls do not share any.  Ids and lengths that
only the device can check are reported in ``status`` (an AkvStatus record, by
default one per device and stream, and one per device for captured calls;
``check=True`` waits and raises BlockOpError, which clears it, and is refused
while capturing).  The tokens
concerned are left out; while the record holds an error, kv_append and
key_bounds write nothing, as the framework's other writes (the reads go on).
That starts with the call that reports it, so any of such a call's other tokens
may be left out as well: append the batch again once the record is clear.
Make a call once before capturing it (a pool's allocator does that for all).
Forward only: an input that asks for a gradient is refused.
"""

from __future__ import annotations

import struct
from functools import lru_cache
from typing import Optional

import torch

from . import _native as N
from .kernels import _as_device_i32, _require_cuda, _status_buffer, raise_for_status, stream_handle

_DTYPES = {torch.float32: N.F32, torch.float16: N.F16, torch.bfloat16: N.BF16}
_GRAPH_STATUS: dict = {}
_COUNTERS: dict = {}
# the C ABI's structs, packed (a tenth of a ctypes.Structure's time, on a path that is all latency)
_POOL = struct.Struct("@Piiiiiiii").pack
_BATCH = struct.Struct("@PPqii").pack
_HEADS = struct.Struct("@Pqq").pack
_capturing = torch._C._cuda_isCurrentStreamCapturing
_current_device = torch._C._cuda_getDevice


def _status(device: torch.device, status: Optional[torch.Tensor], capturing: bool,
            check: bool = False) -> Optional[torch.Tensor]:
    """The caller's status record or the default one.  A captured call uses a
    record of the device that an eager call made (a record made while capturing
    would be cleared by replays of that one graph only); before any, none."""
    if check and capturing:
        raise RuntimeError("check=True waits for the call: not while capturing")
    if status is not None:
        if status.dtype != torch.int32 or status.device != device or status.numel() * 4 < N.STATUS_BYTES:
            raise ValueError("status must be an int32 tensor of 8 elements on the pool's device")
        return status
    if capturing:
        return _GRAPH_STATUS.get(device.index)
    if device.index not in _GRAPH_STATUS:
        _GRAPH_STATUS[device.index] = torch.zeros(N.STATUS_BYTES // 4, dtype=torch.int32, device=device)
    return _status_buffer(device)


def _counters(device: torch.device, stream: int, capturing: bool) -> torch.Tensor:
    """The arrival counters of paged_attention, zero between calls: one
    array per device and stream, and one of its own for a captured call, whose
    replays may overlap other work of any stream."""
    if capturing:
        return torch.zeros(N.ATTENTION_COUNTERS, dtype=torch.int32, device=device)
    key = (device.index, stream)
    buf = _COUNTERS.get(key)
    if buf is None:
        buf = _COUNTERS[key] = torch.zeros(N.ATTENTION_COUNTERS, dtype=torch.int32, device=device)
    return buf


def _no_gradient(x: torch.Tensor, name: str, what: str) -> None:
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: {name} asks for a gradient; this is a forward-only operator")


def _pool_view(pool: torch.Tensor, layer: int, what: str):
    """AkvPagedPool of one layer, and the pool's heads, head_dim and type."""
    shape = pool.shape
    if len(shape) != 6 or shape[2] != 2 or not pool.is_contiguous():
        raise ValueError(f"{what}: pool must be a contiguous "
                         "[blocks, layers, 2, heads, block_size, head_dim] tensor")
    torch_dtype = pool.dtype
    dtype = _DTYPES.get(torch_dtype)
    if dtype is None:
        raise ValueError(f"{what}: pool dtype must be float16, bfloat16 or float32, got {torch_dtype}")
    _no_gradient(pool, "pool", what)
    n, layers, _, heads, bs, dim = shape
    return _POOL(pool.data_ptr(), n, layers, heads, bs, dim, dtype, layer, 0), heads, dim, torch_dtype


def _batch_view(tables, lengths, device: torch.device, what: str):
    """AkvPageBatch, its rows and width, and the tensors it points into."""
    if not (isinstance(tables, torch.Tensor) and tables.dtype == torch.int32 and tables.device == device):
        tables = _as_device_i32(tables, device)
    if not (isinstance(lengths, torch.Tensor) and lengths.dtype == torch.int32 and lengths.device == device):
        lengths = _as_device_i32(lengths, device)
    shape = tables.shape
    if len(shape) != 2 or lengths.dim() != 1 or shape[0] != lengths.shape[0]:
        raise ValueError(f"{what}: tables must be [rows, width] and lengths [rows], got {tuple(tables.shape)} "
                         f"and {tuple(lengths.shape)}")
    rows, width = shape
    stride, step = tables.stride()
    if step != 1 and width > 1:
        tables = tables.contiguous()
        stride = width
    if not lengths.is_contiguous():
        lengths = lengths.contiguous()
    return _BATCH(tables.data_ptr(), lengths.data_ptr(), stride, width, rows), rows, width, tables, lengths


def _heads_view(x: torch.Tensor, dim: int, dtype: torch.dtype, device: torch.device, name: str, what: str) -> bytes:
    """AkvHeads of a [tokens, heads, head_dim] operand of the pool's head_dim, type and device."""
    shape = x.shape
    if len(shape) != 3 or shape[2] != dim:
        raise ValueError(f"{what}: {name} must be [tokens, heads, {dim}], got {tuple(shape)}")
    if x.dtype != dtype or x.device != device:
        raise ValueError(f"{what}: {name} must have the pool's dtype and device ({dtype}, {device}), "
                         f"got {x.dtype}, {x.device}")
    token, head, step = x.stride()
    if step != 1 and dim > 1:
        raise ValueError(f"{what}: {name}'s head_dim must be contiguous")
    _no_gradient(x, name, what)
    return _HEADS(x.data_ptr(), token, head)


def _query_heads(query: torch.Tensor, pool_heads: int, what: str) -> int:
    shape = query.shape
    group, left = divmod(shape[1], pool_heads) if len(shape) == 3 else (0, 1)
    if left or group == 0:
        raise ValueError(f"{what}: query must be [tokens, a multiple of {pool_heads} heads, head_dim], "
                         f"got {tuple(query.shape)}")
    return group


def _span(x: torch.Tensor) -> tuple:
    """Addresses [first, last) that x's elements lie in."""
    if x.numel() == 0:
        return 0, 0
    size = 1 + sum((n - 1) * s for n, s in zip(x.shape, x.stride()))
    return x.data_ptr(), x.data_ptr() + size * x.element_size()


def _apart(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether no element of y shares memory with one of x: their addresses
    do not meet, or do not modulo one of x's strides (views of one buffer
    next to one another in each of its rows, as of a fused projection)."""
    (a, b), (c, d) = _span(x), _span(y)
    if a >= d or c >= b:
        return True
    for period in {n * x.element_size() for n in x.stride() if n > 0}:
        # dimensions whose steps are whole periods stay at one place in it
        ex, ey = (t.element_size() + sum((n - 1) * s * t.element_size() for n, s in zip(t.shape, t.stride())
                                         if n > 1 and s * t.element_size() % period) for t in (x, y))
        at = (c - a) % period
        if at >= ex and at + ey <= period:
            return True
    return False


def _check_output(out: torch.Tensor, like: torch.Tensor, name: str, what: str, *inputs: torch.Tensor) -> None:
    """out has like's shape, no two elements of it share memory, and none
    of it lies within an input."""
    if out.shape != like.shape or out.requires_grad:
        raise ValueError(f"{what}: {name} must be a {tuple(like.shape)} tensor without a gradient")
    if not out.is_contiguous():
        span = 1
        for n, s in sorted(zip(out.shape, out.stride()), key=lambda x: x[1]):
            if n > 1 and s < span:
                raise ValueError(f"{what}: {name}'s elements overlap")
            span += (n - 1) * s
    for x in inputs:
        if not _apart(out, x):
            raise ValueError(f"{what}: {name} shares memory with an input")


def _check_bounds(bounds: torch.Tensor, pool: torch.Tensor, what: str) -> None:
    n, L, _, H, _, D = pool.shape
    if bounds.shape != (n, L, H, 2, D) or bounds.dtype != pool.dtype or bounds.device != pool.device \
            or not bounds.is_contiguous():
        raise ValueError(f"{what}: bounds must be a contiguous {(n, L, H, 2, D)} {pool.dtype} tensor on {pool.device}, "
                         f"got {tuple(bounds.shape)} {bounds.dtype} on {bounds.device}")
    _no_gradient(bounds, "bounds", what)


@lru_cache(maxsize=1024)
def _attention_scratch(geometry: bytes, rows: int, width: int, group: int, keep: int) -> int:
    """Work space of a call, a function of these numbers alone (`geometry`: an
    AkvPagedPool without its address)."""
    n = N.lib.akv_paged_attention_scratch_bytes(bytes(8) + geometry, rows, width, group, keep)
    if n < 0:
        N.check(N.AKV_ERR_INVALID_ARG)
    return n


def _on_device(device: torch.device, call):
    """call() with the pool's device as the current one (a launch goes to the
    current device's context)."""
    if _current_device() == device.index:
        return call()
    with torch.cuda.device(device):
        return call()


def rope_table(rotary_dim: int, positions: int, *, theta: float = 10000.0, inv_freq: Optional[torch.Tensor] = None,
               device="cuda") -> torch.Tensor:
    """The float32 [positions, rotary_dim] table that kv_append takes: the
    cosines of each position's rotary_dim / 2 angles, then their sines, worked
    out in 64 bits.  The frequencies are theta ** (-2 i / rotary_dim), or
    ``inv_freq`` ([rotary_dim / 2], a scaled model's own)."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rope_table: rotary_dim must be positive and even, got {rotary_dim}")
    if inv_freq is None:
        inv_freq = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    if inv_freq.shape != (rotary_dim // 2,):
        raise ValueError(f"rope_table: inv_freq must be [{rotary_dim // 2}], got {tuple(inv_freq.shape)}")
    angles = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv_freq.to(device, torch.float64)
    return torch.cat([angles.cos(), angles.sin()], 1).to(torch.float32)


def kv_append(pool: torch.Tensor, layer: int, key: torch.Tensor, value: torch.Tensor, tables, lengths, *,
              starts: Optional[torch.Tensor] = None, rope: Optional[torch.Tensor] = None, interleaved: bool = False,
              query: Optional[torch.Tensor] = None, query_out: Optional[torch.Tensor] = None,
              bounds: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None,
              check: bool = False) -> Optional[torch.Tensor]:
    """Write a batch's new tokens' keys and values ([tokens, heads, head_dim])
    into layer `layer` of their blocks, in one launch.

    ``lengths`` counts the new tokens in.  With ``starts`` (int32 [rows + 1],
    ascending) row s's new tokens are its last ``starts[s + 1] - starts[s]``,
    held in rows ``starts[s] ..`` of the operands; operand rows behind
    ``starts[-1]`` are padding and nothing is done for them.  Without it
    each row has one new token, row s of the operands (none where its length
    is 0).  No two rows may append to one block: make shared blocks
    exclusive first (ensure_mutable_batch), as for kv_scatter.  The operands do
    not lie in the pool.

    ``rope`` (float32 [positions, rotary_dim], see rope_table) rotates the
    first rotary_dim dimensions of each new key by its position, pairs
    (i, i + rotary_dim / 2), or neighbours with ``interleaved``.  ``query``
    ([tokens, query heads, head_dim]) is rotated the same way and returned
    (in ``query_out`` when given, which may be query itself; rows of padding are
    left as they are there, and undefined without it).  ``bounds``
    ([blocks, layers, heads, 2, head_dim], see key_bounds) is brought up to
    date for the blocks written."""
    what = "kv_append"
    p, H, dim, dtype = _pool_view(pool, layer, what)
    dev = pool.device
    kview, vview = _heads_view(key, dim, dtype, dev, "key", what), _heads_view(value, dim, dtype, dev, "value", what)
    shape = key.shape
    tokens = shape[0]
    if shape[1] != H or value.shape != shape:
        raise ValueError(f"{what}: key and value must be [tokens, {H}, {dim}], got {tuple(shape)} "
                         f"and {tuple(value.shape)}")
    qview = oview = None
    heads = 0
    if query is not None:
        _query_heads(query, H, what)
        qview = _heads_view(query, dim, dtype, dev, "query", what)
        qshape = query.shape
        heads = qshape[1]
        if qshape[0] != tokens:
            raise ValueError(f"{what}: {qshape[0]} queries for {tokens} keys")
        if query_out is None:
            query_out = query.new_empty(qshape)
            oview = _HEADS(query_out.data_ptr(), heads * dim, dim)
        elif query_out is not query:
            same = query_out.data_ptr() == query.data_ptr() and query_out.stride() == query.stride()
            _check_output(query_out, query, "query_out", what, key, value, pool, *(() if same else (query,)))
        if query_out is query:
            _check_output(query_out, query, "query_out", what, key, value, pool)
        if oview is None:
            oview = _heads_view(query_out, dim, dtype, dev, "query_out", what)
    elif query_out is not None:
        raise ValueError(f"{what}: query_out without query")
    rptr, positions, rotary = None, 0, 0
    if rope is not None:
        if rope.dim() != 2 or rope.dtype != torch.float32 or rope.device != dev or not rope.is_contiguous():
            raise ValueError(f"{what}: rope must be a contiguous float32 [positions, rotary_dim] tensor on {dev}")
        _no_gradient(rope, "rope", what)
        if rope.data_ptr() % 16:
            raise ValueError(f"{what}: rope must start on a 16-byte boundary")
        rptr, (positions, rotary) = rope.data_ptr(), rope.shape
    bptr = None
    if bounds is not None:
        _check_bounds(bounds, pool, what)
        bptr = bounds.data_ptr()
    if not pool.is_cuda and not _require_cuda(pool, what):
        return query_out
    b, rows, _, tables, lengths = _batch_view(tables, lengths, dev, what)
    sptr = None
    if starts is not None:
        if not (isinstance(starts, torch.Tensor) and starts.dtype == torch.int32 and starts.device == dev
                and starts.is_contiguous()):
            starts = _as_device_i32(starts, dev)
        if starts.shape != (rows + 1,):
            raise ValueError(f"{what}: starts must be [{rows + 1}], got {tuple(starts.shape)}")
        sptr = starts.data_ptr()

    def call() -> None:
        st = _status(dev, status, _capturing(), check)
        rc = N.lib.akv_kv_append(p, b, kview, vview, tokens, sptr, rptr, positions, rotary, interleaved, qview, oview,
                                 heads, bptr, None if st is None else st.data_ptr(), stream_handle(dev))
        if rc:
            N.check(rc)
        if check and st is not None:
            raise_for_status(st)

    _on_device(dev, call)
    return query_out


def key_bounds(pool: torch.Tensor, layer: int, tables, lengths, bounds: Optional[torch.Tensor] = None, *,
               status: Optional[torch.Tensor] = None, check: bool = False) -> torch.Tensor:
    """Write the bounds of every block that the batch's rows hold, from the
    keys in layer `layer`: ``bounds[b, layer, h]`` gets the minimum and the
    maximum, by dimension, of block b's keys (of a row's last block, those
    that the row holds).  Makes the [blocks, layers, heads, 2, head_dim]
    tensor (zeros elsewhere) when none is given.  kv_append keeps bounds up to date by
    itself; this is for blocks that were written by other means.  Rows that
    share a block hold equally many of its keys: of rows with one table and other
    lengths (several new tokens of a sequence) give the longest alone."""
    what = "key_bounds"
    p = _pool_view(pool, layer, what)[0]
    n, L, _, H, _, D = pool.shape
    if bounds is None:
        bounds = torch.zeros((n, L, H, 2, D), dtype=pool.dtype, device=pool.device)
    else:
        _check_bounds(bounds, pool, what)
    if not _require_cuda(pool, what):
        return bounds
    dev = pool.device
    b, _, _, tables, lengths = _batch_view(tables, lengths, dev, what)

    def call() -> None:
        st = _status(dev, status, _capturing(), check)
        N.check(N.lib.akv_key_bounds(p, b, bounds.data_ptr(), None if st is None else st.data_ptr(),
                                     stream_handle(dev)))
        if check and st is not None:
            raise_for_status(st)

    _on_device(dev, call)
    return bounds


def select_blocks(query: torch.Tensor, bounds: torch.Tensor, layer: int, tables, lengths, keep: int, *,
                  block_size: int, first: int = 1, last: int = 1, status: Optional[torch.Tensor] = None,
                  check: bool = False) -> torch.Tensor:
    """The `keep` blocks of each row that matter most to its new token, for
    each key head: int32 [rows, heads, keep], ascending places in the row's
    table, -1 behind them where a row holds fewer.

    A row of no more than `keep` blocks keeps all.  Else it keeps its `first`
    first and `last` last blocks and, of the others, those of the highest
    score: the sum, over the query heads that share the key head, of the
    highest score that a key within the block's ``bounds`` could have.  Of
    equal scores the lower place is taken; a NaN score counts as the highest (an
    infinite bound makes one where no query head of the group has the sign that meets it)."""
    what = "select_blocks"
    if bounds.dim() != 5 or bounds.shape[3] != 2 or not bounds.is_contiguous():
        raise ValueError(f"{what}: bounds must be a contiguous [blocks, layers, heads, 2, head_dim] tensor")
    n, L, H, _, D = bounds.shape
    dtype = _DTYPES.get(bounds.dtype)
    if dtype is None:
        raise ValueError(f"{what}: bounds dtype must be float16, bfloat16 or float32, got {bounds.dtype}")
    _no_gradient(bounds, "bounds", what)
    keep, first, last = int(keep), int(first), int(last)
    if keep < 1 or first < 0 or last < 0 or first + last > keep:
        raise ValueError(f"{what}: needs keep >= 1 and 0 <= first + last <= keep, got {keep}, {first}, {last}")
    dev = bounds.device
    group = _query_heads(query, H, what)
    qview = _heads_view(query, D, bounds.dtype, dev, "query", what)
    rows = query.shape[0]
    selected = query.new_empty((rows, H, keep), dtype=torch.int32)
    if not bounds.is_cuda and not _require_cuda(bounds, what):
        return selected
    p = _POOL(0, n, L, H, block_size, D, dtype, layer, 0)
    b, batch, width, tables, lengths = _batch_view(tables, lengths, dev, what)
    if batch != rows:
        raise ValueError(f"{what}: {rows} queries for {batch} rows")

    def call() -> None:
        st = _status(dev, status, _capturing(), check)
        scratch = query.new_empty(max(0, N.lib.akv_select_blocks_scratch_bytes(rows, H, width, keep)),
                                  dtype=torch.uint8)
        rc = N.lib.akv_select_blocks(p, bounds.data_ptr(), b, qview, group, keep, first, last, selected.data_ptr(),
                                     scratch.data_ptr(), scratch.numel(), None if st is None else st.data_ptr(),
                                     stream_handle(dev))
        if rc:
            N.check(rc)
        if check and st is not None:
            raise_for_status(st)

    _on_device(dev, call)
    return selected


def paged_attention(query: torch.Tensor, pool: torch.Tensor, layer: int, tables, lengths, *,
                    scale: Optional[float] = None, window: int = 0, selected: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None, return_lse: bool = False,
                    status: Optional[torch.Tensor] = None, check: bool = False):
    """Attention of one new token per row over layer `layer` of the row's
    blocks: query and the result are [rows, heads, head_dim] with a multiple
    of the pool's heads (query head i reads key head i // group), in the
    pool's type.

    Positions below the row's length take part; with ``window`` > 0 only the
    last `window` of them (blocks wholly before them may have been freed);
    with ``selected`` (int32 [rows, kv heads, keep], distinct places in the
    row's table, the valid ones first, then -1; see select_blocks) only those
    of the selected blocks.  ``scale`` defaults to head_dim ** -0.5.  A row with no position gives 0.
    With ``return_lse`` also the float32 [rows, heads] natural
    logarithm of each softmax's sum (-inf for an empty row).  Several new
    tokens of one sequence are several rows with the same table and
    their own lengths.  NaN and infinities in blocks that a row does not read, or behind
    its last position, do not reach it; an infinite value among those that
    take part makes its dimension infinite or NaN (a weight is held as a sum
    of two 16-bit numbers, and infinity times either may be NaN)."""
    what = "paged_attention"
    p, kv_heads, dim, dtype = _pool_view(pool, layer, what)
    dev = pool.device
    group = _query_heads(query, kv_heads, what)
    qview = _heads_view(query, dim, dtype, dev, "query", what)
    rows, heads, _ = query.shape
    if out is None:
        out = query.new_empty((rows, heads, dim))
        oview = _HEADS(out.data_ptr(), heads * dim, dim)
    else:
        _check_output(out, query, "out", what, query, pool)
        oview = _heads_view(out, dim, dtype, dev, "out", what)
    lse = query.new_empty((rows, heads), dtype=torch.float32) if return_lse else None
    if not pool.is_cuda and not _require_cuda(pool, what):
        return (out, lse) if return_lse else out
    window = int(window)
    if window < 0:
        raise ValueError(f"{what}: window must not be negative, got {window}")
    b, batch, width, tables, lengths = _batch_view(tables, lengths, dev, what)
    if batch != rows:
        raise ValueError(f"{what}: {rows} queries for {batch} rows")
    sel, keep = None, 0
    if selected is not None:
        keep = selected.shape[-1] if selected.dim() == 3 else 0
        if selected.shape != (rows, kv_heads, keep) or keep == 0 or selected.dtype != torch.int32 \
                or selected.device != dev or not selected.is_contiguous():
            raise ValueError(f"{what}: selected must be a contiguous int32 [{rows}, {kv_heads}, keep] tensor "
                             f"on {dev}")
        sel = selected.data_ptr()

    def call() -> None:
        capturing = _capturing()
        st, stream = _status(dev, status, capturing, check), stream_handle(dev)
        scratch = query.new_empty(_attention_scratch(p[8:], rows, width, group, keep), dtype=torch.uint8)
        rc = N.lib.akv_paged_attention(
            p, b, qview, group, dim ** -0.5 if scale is None else scale, min(window, (1 << 31) - 1), sel, keep, oview,
            None if lse is None else lse.data_ptr(), scratch.data_ptr(), scratch.numel(),
            _counters(dev, stream, capturing).data_ptr(), None if st is None else st.data_ptr(), stream)
        if rc:
            N.check(rc)
        if check and st is not None:
            raise_for_status(st)

    _on_device(dev, call)
    return (out, lse) if return_lse else out
