"""Which tensors attention's operators take as outputs beside their inputs:
views of one buffer that share no element are apart, others are not."""

import itertools
import random

import pytest
import torch

from agentkv_b200 import _native as N
from agentkv_b200 import attention as A


def _addresses(x):
    at = torch.zeros(1, dtype=torch.int64)
    for n, s in zip(x.shape, x.stride()):
        at = (at[:, None] + torch.arange(n) * s).reshape(-1)
    return {x.data_ptr() + int(i) * x.element_size() + b for i in at for b in range(x.element_size())}


@pytest.mark.parametrize("tokens", [1, 2, 5])
def test_views_of_a_fused_projection_are_apart(tokens):
    Hq, H, D = 6, 2, 8
    packed = torch.zeros(tokens, Hq + 2 * H, D, dtype=torch.bfloat16)       # [tokens, all heads, head_dim]
    q, k, v = packed[:, :Hq], packed[:, Hq:Hq + H], packed[:, Hq + H:]
    third = torch.zeros(tokens, 3, H, D, dtype=torch.float16).unbind(1)       # [tokens, (q, k, v), heads, head_dim]
    by_head = torch.zeros(tokens, H, 3, D, dtype=torch.float32).unbind(2)     # [tokens, heads, (q, k, v), head_dim]
    by_dim = torch.zeros(tokens, H, 3 * D, dtype=torch.float32).split(D, 2)   # [tokens, heads, (q, k, v) of head_dim]
    heads_first = torch.zeros(3, H, tokens, D).transpose(1, 2).unbind(0)      # (q, k, v) of [heads, tokens, head_dim]
    for views in ((q, k, v), third, by_head, by_dim, heads_first):
        for x, y in itertools.permutations(views, 2):
            assert A._apart(x, y)
            A._check_output(x, x, "query_out", "kv_append", y)
    for x, y in ((q, packed[:, Hq - 1:Hq + 1]), (k, packed[:, :Hq + 1]), (v, packed), (packed, v), (q, q)):
        assert not A._apart(x, y)
        with pytest.raises(ValueError, match="shares memory"):
            A._check_output(x, x, "query_out", "kv_append", y)


def test_no_overlap_is_missed():
    """Random views of one buffer against their elements' addresses: what is
    called apart has none in common."""
    rng = random.Random(5)
    buf = torch.zeros(4000, dtype=torch.float16)
    called = met = 0
    for _ in range(4000):
        views = []
        for _ in range(2):
            shape = [rng.randint(1, 5), rng.randint(1, 4), rng.choice([1, 2, 3, 4])]
            stride = [rng.choice([0, 4, 8, 12, 16, 24, 30]), rng.choice([0, 2, 4, 8, 16]), 1]
            x = buf[rng.randint(0, 60):].as_strided(shape, stride, rng.randint(0, 60))
            views.append(x.view(torch.bfloat16) if rng.random() < 0.3 else x)
        common = bool(_addresses(views[0]) & _addresses(views[1]))
        apart = A._apart(*views)
        assert not (apart and common), [(x.shape, x.stride(), x.storage_offset()) for x in views]
        called += apart
        met += not common
    assert called > 0.6 * met  # and it is not all refused


@pytest.mark.parametrize("dtype", [N.F32, N.F16, N.BF16])
def test_the_work_space_is_enough_for_every_alignment(dtype):
    """The size does not depend on the addresses, the engine does: a call of exactly that
    size is refused for its missing counters alone."""
    rng = random.Random(dtype)
    size = 4 if dtype == N.F32 else 2
    for dim in [1, 2, 4, 7, 8, 12, 56, 60, 64, 68, 72, 80, 96, 100, 104, 128, 130, 132, 136, 200, 204, 252, 256]:
        for group in [1, 2, 3, 4, 5, 8, 9, 16, 17]:
            rows, width, keep, bs = rng.choice([1, 3, 200]), rng.choice([1, 7, 500]), rng.choice([0, 2]), 16
            geometry = (64, 2, 2, bs, dim, dtype, 0, 0)
            need = N.lib.akv_paged_attention_scratch_bytes(A._POOL(0, *geometry), rows, width, group, keep)
            assert need > 0
            for at in (1 << 20, (1 << 20) + 8, (1 << 20) + 4, (1 << 20) + size):
                heads = A._HEADS(at, 2 * group * dim, dim)
                batch = A._BATCH(1 << 20, 1 << 20, width, width, rows)
                rc = N.lib.akv_paged_attention(A._POOL(1 << 20, *geometry), batch, heads, group, 1.0, 0,
                                               1 << 20 if keep else None, keep, heads, None, 1 << 20, need, None, None, None)
                assert rc == N.AKV_ERR_INVALID_ARG and "counters" in N.last_error(), (dim, group, at, N.last_error())


def _meta(*shape, dtype=torch.bfloat16, **kw):
    return torch.empty(shape, dtype=dtype, device="meta", **kw)


def test_every_input_that_asks_for_a_gradient_is_refused():
    pool, asks = _meta(8, 2, 2, 2, 16, 64), _meta(8, 2, 2, 2, 16, 64, requires_grad=True)
    bounds, asks_b = _meta(8, 2, 2, 2, 64), _meta(8, 2, 2, 2, 64, requires_grad=True)
    q, k = _meta(3, 4, 64), _meta(3, 2, 64)
    calls = [
        ("pool", lambda: A.paged_attention(q, asks, 0, None, None)),
        ("pool", lambda: A.kv_append(asks, 0, k, k, None, None)),
        ("pool", lambda: A.key_bounds(asks, 0, None, None)),
        ("bounds", lambda: A.key_bounds(pool, 0, None, None, asks_b)),
        ("bounds", lambda: A.kv_append(pool, 0, k, k, None, None, bounds=asks_b)),
        ("bounds", lambda: A.select_blocks(q, asks_b, 0, None, None, 5, block_size=16)),
        ("rope", lambda: A.kv_append(pool, 0, k, k, None, None, rope=_meta(9, 64, dtype=torch.float32, requires_grad=True))),
    ]
    for name, call in calls:
        with pytest.raises(ValueError, match=f"{name} asks for a gradient"):
            call()
        with torch.no_grad():
            call()
    A.select_blocks(q, bounds, 0, None, None, 5, block_size=16)
