"""DecodeBatch — a set of agents decoding together on the pool's own pages.

The reference's consumers hold one cache per agent and assemble its K and V
for every layer (agentkv/hf_cache.py:57-153).  A DecodeBatch holds the block
tables and lengths of many agents on the device, and a step of all of them is
one ``advance`` (blocks allocated, shared ones copied on write, tables
uploaded) and per layer one ``append`` and one ``attend``:

    batch = pool.decode_batch([pool.fork(root) for _ in range(64)])
    batch.advance([[t] for t in next_tokens])
    for layer in range(num_layers):
        q = batch.append(layer, k, v, query=q, rope=rope)   # k, v: [64, kv_heads, head_dim]
        out = batch.attend(layer, q)                        # [64, heads, head_dim]

The device tensors keep their addresses while the rows and the width do (give
``width`` to hold it), so the calls of a step can be captured once and
replayed after each ``advance``: a step captured after one of one token each
serves such steps, one captured after an uneven one (operands with rows for
the most tokens) any.
"""

from __future__ import annotations

from typing import List, Optional, Sequence

import numpy as np
import torch

from . import _native as N
from . import attention as A
from . import kernels as K
from .radix_tree import NodeHandle


class DecodeBatch:
    """The agents `handles` of `pool`, whose tokens so far have their keys and
    values in the pool, in that order; rows behind them, up to `rows`, are padding.
    ``width`` is the blocks that a row's table has room for (grown as
    needed when None).  With ``bounds`` (True, or a tensor that several
    batches of the pool share; see attention.key_bounds) ``append`` keeps the
    blocks' key bounds, which ``attend(keep=...)`` ranks them by; a new tensor
    starts with the bounds of the blocks that the agents hold.

    What only the device can see goes to the batch's own record, ``status``
    (captured calls' too): ``check()`` waits for it and raises, and ``advance``
    raises, before anything changes, what has come back by then of earlier steps
    (whose appends from the refused one on have written nothing)."""

    def __init__(self, pool, handles: Sequence[NodeHandle], *, rows: Optional[int] = None, width: Optional[int] = None,
                 bounds=None) -> None:
        self.pool = pool
        self.handles: List[NodeHandle] = list(handles)
        n = len(self.handles)
        self.rows = n if rows is None else int(rows)
        if self.rows < n:
            raise ValueError(f"DecodeBatch: {n} agents in {self.rows} rows")
        if len({h.handle_id for h in self.handles}) != n:
            raise ValueError("DecodeBatch: an agent appears twice")
        self._fixed = width is not None
        data = pool._allocator._kv_data
        self._data = data
        ids = [pool.get_block_ids(h) for h in self.handles]
        self._all_held([len(b) for b in ids])
        need = max([len(b) for b in ids], default=0)
        self.width = max(1, need) if width is None else int(width)
        self.tables = torch.zeros((self.rows, self.width), dtype=torch.int32, device=data.device)
        self.lengths = torch.zeros(self.rows, dtype=torch.int32, device=data.device)
        self.starts: Optional[torch.Tensor] = None  # of the last advance, when a row got more or less than one token
        self._starts: Optional[torch.Tensor] = None  # where they lie, from the first such advance on
        self._advanced = False  # the last advance's new tokens are there to be appended
        self._positions = 0  # what the longest row that got new tokens holds
        self.status = torch.zeros(N.STATUS_BYTES // 4, dtype=torch.int32, device=data.device)
        self._seen = torch.zeros(N.STATUS_BYTES // 4, dtype=torch.int32, pin_memory=data.is_cuda)
        self._upload(ids)
        self.bounds: Optional[torch.Tensor] = None
        if bounds is not None and bounds is not False:
            if bounds is True:
                n_blocks, layers, _, heads, _, dim = data.shape
                self.bounds = torch.zeros((n_blocks, layers, heads, 2, dim), dtype=data.dtype, device=data.device)
                for layer in range(layers):
                    A.key_bounds(data, layer, self.tables, self.lengths, self.bounds, status=self.status)
            else:
                A._check_bounds(bounds, data, "DecodeBatch")
                self.bounds = bounds

    def _all_held(self, blocks: Sequence[int]) -> None:
        """Refuses an agent whose tokens are more than its blocks hold (a root
        made of a prompt that is not in the pool yet)."""
        bs = self.pool.block_size
        for h, n in zip(self.handles, blocks):
            if len(h.tokens) > n * bs:
                raise ValueError(f"DecodeBatch: an agent has {len(h.tokens)} tokens in {n} blocks of {bs}")

    def _upload(self, ids: List[List[int]]) -> None:
        need = max([len(b) for b in ids], default=0)
        if need > self.width:
            if self._fixed:
                raise ValueError(f"DecodeBatch: a table of {self.width} blocks cannot hold {need}")
            self.width = max(need, 2 * self.width)
            self.tables = torch.zeros((self.rows, self.width), dtype=torch.int32, device=self.tables.device)
        table = np.zeros((self.rows, self.width), np.int32)
        for i, b in enumerate(ids):
            table[i, : len(b)] = b
        lens = np.zeros(self.rows, np.int32)
        lens[: len(self.handles)] = [len(h.tokens) for h in self.handles]
        # (from pageable memory: the copy has left these arrays when it returns)
        self.tables.copy_(torch.from_numpy(table))
        self.lengths.copy_(torch.from_numpy(lens))

    def check(self) -> None:
        """Wait for the calls so far and raise BlockOpError for the first that
        the device refused, if any (which clears it)."""
        self._seen.zero_()
        if self.status.is_cuda:
            K.raise_for_status(self.status)

    def advance(self, tokens: Sequence[Sequence[int]]) -> None:
        """Give agent i the new tokens ``tokens[i]`` (none: it sits this step
        out): room is allocated, blocks that the new tokens go to are made
        exclusive (copied when shared), and tables and lengths uploaded.  The
        keys and values follow by ``append``, for every layer."""
        if len(tokens) != len(self.handles):
            raise ValueError(f"DecodeBatch.advance: tokens for {len(tokens)} of {len(self.handles)} agents")
        pool, bs = self.pool, self.pool.block_size
        self._advanced = False
        if self._seen[0]:
            self.check()
        counts = [len(t) for t in tokens]
        held = [len(pool.get_block_ids(h)) for h in self.handles]  # refuses a freed agent before anything changes
        self._all_held(held)
        if self._fixed:
            for h, n in zip(self.handles, counts):
                if len(h.tokens) + n > self.width * bs:
                    raise ValueError(f"DecodeBatch: a table of {self.width} blocks cannot hold "
                                     f"{len(h.tokens) + n} tokens")
        writes = []
        for h, n in zip(self.handles, counts):
            if n == 0:
                continue
            first, shared = len(h.tokens) // bs, h.shared_match_len // bs
            last = (len(h.tokens) + n - 1) // bs
            if first < shared:
                raise RuntimeError("Cannot overwrite shared prefix blocks!")
            writes += [(h, b - shared) for b in range(first, last + 1)]
        for h, n, blocks in zip(self.handles, counts, held):
            if n:
                required = (len(h.tokens) + n + bs - 1) // bs - blocks
                if required > 0:
                    pool.allocate_blocks(h, required)
        if writes:
            pool.ensure_mutable_batch(writes)
        for h, n, new in zip(self.handles, counts, tokens):
            if n:
                pool.append_tokens(h, list(new))
        self._upload([pool.get_block_ids(h) for h in self.handles])
        even = all(n == 1 for n in counts)
        if not even and self._starts is None:
            self._starts = torch.zeros(self.rows + 1, dtype=torch.int32, device=self.lengths.device)
        if self._starts is not None:  # (kept right in even steps too: a captured uneven one reads them)
            starts = np.zeros(self.rows + 1, np.int32)
            starts[1 : len(counts) + 1] = np.cumsum(counts)
            starts[len(counts) + 1 :] = starts[len(counts)]
            self._starts.copy_(torch.from_numpy(starts))
        self.starts = None if even else self._starts
        self._positions = max([len(h.tokens) for h, n in zip(self.handles, counts) if n], default=0)
        if self.status.is_cuda:
            self._seen.copy_(self.status, non_blocking=True)
        self._advanced = True

    def append(self, layer: int, key: torch.Tensor, value: torch.Tensor, **kw) -> Optional[torch.Tensor]:
        """attention.kv_append of the last advance's new tokens, all agents'
        behind one another: key and value [tokens, kv_heads, head_dim] (where
        each agent got one token: of the agents, or of all rows, padding
        among them); ``query``, ``rope`` and the rest as there.  Returns the
        rotated queries, if any.  Refused before an advance and behind one that failed."""
        if not self._advanced:
            raise RuntimeError("DecodeBatch.append: no new tokens; advance() comes first")
        rope = kw.get("rope")
        if rope is not None and rope.shape[0] < self._positions:
            raise ValueError(f"DecodeBatch.append: a rope table of {rope.shape[0]} positions for {self._positions} tokens")
        kw.setdefault("status", self.status)
        tables, lengths, n = self.tables, self.lengths, len(self.handles)
        if self.starts is None and key.shape[0] == n < self.rows:
            tables, lengths = tables[:n], lengths[:n]
        return A.kv_append(self._data, layer, key, value, tables, lengths, starts=self.starts, bounds=self.bounds, **kw)

    def attend(self, layer: int, query: torch.Tensor, *, keep: int = 0, first: int = 1, last: int = 1, **kw):
        """attention.paged_attention of one query per row, [rows, heads,
        head_dim], over the row's tokens; with ``keep`` over the `keep` blocks
        that attention.select_blocks picks (needs the batch's bounds)."""
        kw.setdefault("status", self.status)
        if keep:
            if self.bounds is None:
                raise ValueError("DecodeBatch.attend: keep needs a batch with bounds")
            kw["selected"] = A.select_blocks(query, self.bounds, layer, self.tables, self.lengths, keep,
                                             block_size=self.pool.block_size, first=first, last=last,
                                             status=kw["status"])
        return A.paged_attention(query, self._data, layer, self.tables, self.lengths, **kw)
