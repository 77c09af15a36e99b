"""The paged operators where calls go wrong or values leave the ordinary range:
batches with bad rows, scores far apart, agents on a matched prefix, captured
calls whose inputs move on."""

import math

import pytest
import torch

from agentkv_b200 import AgentKVPool, PoolConfig
from agentkv_b200 import _native as N
from agentkv_b200 import attention as A
from agentkv_b200 import kernels as K

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, dtype):
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


# ── append: rows that are reported while others are written ──────────────────
@pytest.mark.parametrize("kind", ["table", "rope", "starts"])
def test_ragged_append_with_bad_rows_writes_right_words_or_none(kind):
    """Bad rows among many: they are reported, and of every other token each
    word is either the right one or as it was, in its own block only.  CTAs of the
    launch read the record while others report into it."""
    H, G, D, bs, rows = 2, 2, 64, 4, 400
    g = _gen(3)
    old = [(7 * s) % 23 for s in range(rows)]
    new = [1 + (5 * s) % 9 for s in range(rows)]
    need = [-(-(o + n) // bs) for o, n in zip(old, new)]
    W, total = max(need) + 1, sum(need)
    table, at = torch.zeros((rows, W), dtype=torch.int32), 0
    for s in range(rows):
        table[s, :need[s]] = torch.arange(at, at + need[s], dtype=torch.int32)
        at += need[s]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    T = starts[-1]
    lengths = [o + n for o, n in zip(old, new)]
    bad = set(range(3, rows, 41))
    given, positions = list(starts), 64
    if kind == "table":
        for s in bad:
            table[s, old[s] // bs] = (-1, total, 2 ** 31 - 1)[s % 3]
    elif kind == "rope":
        positions = 28
        bad = {s for s in range(rows) if lengths[s] > positions}
        assert 0 < len(bad) < rows // 4
    else:  # one start out of range spoils the row before it and the row behind it
        for s in bad:
            given[s] = (-1, T + 1)[s % 2]
        bad |= {s - 1 for s in bad}
    table, lens = table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)
    dev_starts = torch.tensor(given, dtype=torch.int32, device=DEV)
    rope = A.rope_table(D, positions, device=DEV)
    good_rope = A.rope_table(D, 64, device=DEV)
    good_table = torch.zeros((rows, W), dtype=torch.int32)
    at = 0
    for s in range(rows):
        good_table[s, :need[s]] = torch.arange(at, at + need[s], dtype=torch.int32)
        at += need[s]
    k, v = (_randn(g, T, H, D, dtype=BF16) for _ in range(2))
    q = _randn(g, T, H * G, D, dtype=BF16)
    before = _randn(g, total, 1, 2, H, bs, D, dtype=BF16)
    b0 = torch.full((total, 1, H, 2, D), 9.0, dtype=BF16, device=DEV)
    right, rb, rq = before.clone(), b0.clone(), torch.full_like(q, 3.0)
    A.kv_append(right, 0, k, v, good_table, lens, starts=starts, rope=good_rope, query=q, query_out=rq, bounds=rb,
                check=True)
    owner = torch.zeros(total, dtype=torch.long)
    for s in range(rows):
        owner[good_table[s, :need[s]].long()] = s
    is_bad = torch.zeros(rows, dtype=torch.bool)
    is_bad[list(bad)] = True
    spoilt = is_bad[owner].to(DEV)
    token_bad = torch.repeat_interleave(is_bad, torch.tensor(new)).to(DEV)
    for _ in range(25):
        pool, bounds, qo = before.clone(), b0.clone(), torch.full_like(q, 3.0)
        st = torch.zeros(8, dtype=torch.int32, device=DEV)
        A.kv_append(pool, 0, k, v, table, lens, starts=dev_starts, rope=rope, query=q, query_out=qo, bounds=bounds,
                    status=st)
        code, row = K.read_status(st)[:2]
        assert code == N.AKV_ERR_OUT_OF_RANGE and row in bad
        assert ((pool == before) | (pool == right)).all()
        assert ((bounds == b0) | (bounds == rb)).all()
        assert ((qo == 3.0) | (qo == rq)).all()
        if kind == "starts":  # no token of such a row is known
            assert torch.equal(pool[spoilt], before[spoilt]) and torch.equal(bounds[spoilt], b0[spoilt])
            assert (qo[token_bad] == 3.0).all()
    # and whole again once the record is clear
    pool, bounds, qo = before.clone(), b0.clone(), torch.full_like(q, 3.0)
    A.kv_append(pool, 0, k, v, good_table, lens, starts=starts, rope=good_rope, query=q, query_out=qo, bounds=bounds,
                check=True)
    assert torch.equal(pool, right) and torch.equal(bounds, rb) and torch.equal(qo, rq)
