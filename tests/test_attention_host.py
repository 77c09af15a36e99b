"""agentkv_b200.attention without a GPU: the dealing and joining of
paged_attention's work (a model of its index arithmetic), the checks of
arguments in Python and behind the C ABI, and the tables of angles."""

import ctypes as C
import math
import random

import pytest
import torch

import attend_model as M
from agentkv_b200 import _native as N
from agentkv_b200 import attention as A


@pytest.mark.parametrize("seed", range(6))
def test_every_chunk_is_read_once_and_every_piece_joined(seed):
    rng = random.Random(seed)
    for _ in range(300):
        bs = rng.choice([1, 2, 4, 8, 16, 64, 256])
        width = rng.randint(1, max(2, 1500 // bs))
        most = width * bs
        lengths = [rng.choice([-1, 0, 1, most, most + 3, rng.randint(0, most)]) for _ in range(rng.randint(1, 14))]
        heads, parts = rng.randint(1, 4), rng.randint(1, 3)
        window, keep = rng.choice([0, 0, 1, 100, most]), rng.choice([0, 0, 1, 5])
        reads, _ = M.simulate(lengths, width, bs, heads, parts, rng.choice([1, 2, 7, 148, 444]), window, keep)
        assert len(set(reads)) == len(reads)
        want = {(s, h, p, c) for s, n in enumerate(lengths) for _, _, f, k in [M.extent(n, width, bs, window, keep)]
                for h in range(heads) for p in range(parts) for c in range(f, f + k)}
        assert set(reads) == want


def test_two_levels_of_joining():
    """One pair over every CTA of the largest grid."""
    reads, joins = M.simulate([592 * 2 * 64], 592 * 8, 16, 1, 1, 592)
    assert len(reads) == 1184 and sorted(joins[(0, 0)]) == list(range(592))
    assert 3 * 592 <= N.ATTENTION_COUNTERS


@pytest.mark.parametrize("count", [1, 8])
def test_positions_that_take_part(count):
    for n in range(0, 20):
        for lo in range(0, n + 1):
            for pos in range(0, 24):
                want = sum(1 << i for i in range(count) if lo <= pos + i < n)
                assert M.taking_part(n, lo, pos, count) == want


# ── the C ABI refuses before it touches the GPU ──────────────────────────────
def _pool(**kw):
    v = dict(data=1 << 20, n=64, layers=2, heads=8, bs=16, dim=128, dtype=N.BF16, layer=1)
    v.update(kw)
    return A._POOL(v["data"], v["n"], v["layers"], v["heads"], v["bs"], v["dim"], v["dtype"], v["layer"], 0)


def _batch(tables=1 << 20, lengths=1 << 20, stride=4, width=4, rows=3):
    return A._BATCH(tables, lengths, stride, width, rows)


def _heads(data=1 << 20, token=1024, head=128):
    return A._HEADS(data, token, head)


def _attend(pool=None, batch=None, query=None, group=4, window=0, selected=None, keep=0, out=None, scratch=1 << 20,
            nbytes=1 << 30, counters=1 << 20):
    return N.lib.akv_paged_attention(pool or _pool(), batch or _batch(), query or _heads(), group, 1.0, window, selected,
                                     keep, out or _heads(), None, scratch, nbytes, counters, None, None)


def test_packed_structs_have_the_header_s_layout():
    for packed, struct in ((_pool(), N.AkvPagedPool), (_batch(), N.AkvPageBatch), (_heads(), N.AkvHeads)):
        assert len(packed) == C.sizeof(struct)
    p = N.AkvPagedPool.from_buffer_copy(_pool(layer=1, dim=96))
    assert (p.data, p.total_blocks, p.num_layers, p.num_kv_heads, p.block_size, p.head_dim, p.dtype, p.layer) \
        == (1 << 20, 64, 2, 8, 16, 96, N.BF16, 1)
    b = N.AkvPageBatch.from_buffer_copy(_batch(stride=7, width=5, rows=2))
    assert (b.table_stride, b.table_width, b.rows) == (7, 5, 2)


@pytest.mark.parametrize("kw", [
    dict(pool=dict(n=0)), dict(pool=dict(bs=12)), dict(pool=dict(bs=0)), dict(pool=dict(dim=257)),
    dict(pool=dict(dim=0)), dict(pool=dict(layer=2)), dict(pool=dict(layer=-1)), dict(pool=dict(dtype=3)),
    dict(pool=dict(data=(1 << 20) + 1)), dict(pool=dict(data=0)), dict(pool=dict(heads=0)),
    dict(batch=dict(rows=-1)), dict(batch=dict(width=-1)), dict(batch=dict(tables=0)), dict(batch=dict(lengths=0)),
    dict(batch=dict(width=1 << 27, rows=1)), dict(query=dict(data=0)), dict(query=dict(token=-1)),
    dict(query=dict(data=(1 << 20) + 1)), dict(out=dict(data=0)), dict(out=dict(head=-1)), dict(group=0), dict(window=-1),
    dict(group=1 << 29), dict(selected=1 << 20, keep=0), dict(scratch=0), dict(nbytes=16), dict(counters=0),
    dict(scratch=(1 << 20) + 4),
])
def test_attention_refuses(kw):
    kw = {k: {"pool": _pool, "batch": _batch, "query": _heads, "out": _heads}[k](**v) if isinstance(v, dict) else v
          for k, v in kw.items()}
    assert _attend(**kw) == N.AKV_ERR_INVALID_ARG
    assert "akv_paged_attention" in N.last_error()


def test_attention_of_no_rows_needs_nothing():
    assert _attend(batch=_batch(rows=0), scratch=0, nbytes=0, counters=0) == N.AKV_OK


def test_scratch_does_not_grow_with_the_batch_for_ever():
    one = A._attention_scratch(_pool()[8:], 1, 1, 4, 0)
    many = A._attention_scratch(_pool()[8:], 4096, 4096, 4, 0)
    assert 0 < one < many == A._attention_scratch(_pool()[8:], 8192, 8192, 4, 0)
    with pytest.raises(N.NativeError):
        A._attention_scratch(_pool(dim=300)[8:], 1, 1, 4, 0)


@pytest.mark.parametrize("kw", [
    dict(tokens=-1), dict(tokens=2), dict(rotary=3), dict(rotary=0), dict(rotary=130), dict(rope=(1 << 20) + 4),
    dict(key=dict(data=0)), dict(value=dict(token=-1)), dict(qheads=-1), dict(query=dict(data=0)),
    dict(bounds=(1 << 20) + 1), dict(pool=dict(bs=24)),
])
def test_append_refuses(kw):
    tokens = kw.get("tokens", 3)
    made = {k: {"pool": _pool, "key": _heads, "value": _heads, "query": _heads}[k](**v) for k, v in kw.items()
            if isinstance(v, dict)}
    rc = N.lib.akv_kv_append(made.get("pool") or _pool(), _batch(), made.get("key") or _heads(),
                             made.get("value") or _heads(), tokens, None, kw.get("rope", 1 << 20), 100,
                             kw.get("rotary", 128), 0, made.get("query") or _heads(), _heads(), kw.get("qheads", 32),
                             kw.get("bounds", 1 << 20), None, None)
    assert rc == N.AKV_ERR_INVALID_ARG and "akv_kv_append" in N.last_error()


@pytest.mark.parametrize("kw", [dict(keep=0), dict(first=-1), dict(first=5, last=4), dict(group=0), dict(nbytes=8),
                                dict(bounds=0), dict(selected=0)])
def test_select_refuses(kw):
    v = dict(keep=3, first=1, last=1, group=4, nbytes=1 << 30, bounds=1 << 20, selected=1 << 20)
    v.update(kw)
    rc = N.lib.akv_select_blocks(_pool(data=0), v["bounds"], _batch(), _heads(), v["group"], v["keep"], v["first"],
                                 v["last"], v["selected"], 1 << 20, v["nbytes"], None, None)
    assert rc == N.AKV_ERR_INVALID_ARG and "akv_select_blocks" in N.last_error()
    assert N.lib.akv_select_blocks_scratch_bytes(4, 8, 100, 100) == 0  # nothing to rank
    assert N.lib.akv_select_blocks_scratch_bytes(4, 8, 101, 100) > 0
    assert N.lib.akv_select_blocks_scratch_bytes(4, 8, 101, 0) == -1


# ── the checks in Python, on tensors without bytes ──────────────────────────
def _meta(*shape, dtype=torch.bfloat16, **kw):
    return torch.empty(shape, dtype=dtype, device="meta", **kw)


POOL = (64, 2, 2, 8, 16, 128)


def _call(query=None, pool=None, tables=None, lengths=None, **kw):
    return A.paged_attention(_meta(3, 32, 128) if query is None else query, _meta(*POOL) if pool is None else pool, 1,
                             _meta(3, 4, dtype=torch.int32), _meta(3, dtype=torch.int32), **kw)


def test_meta_pools_return_shapes():
    out, lse = _call(return_lse=True)
    assert out.shape == (3, 32, 128) and lse.shape == (3, 32) and lse.dtype == torch.float32
    bounds = A.key_bounds(_meta(*POOL), 0, None, None)
    assert bounds.shape == (64, 2, 8, 2, 128) and bounds.dtype == torch.bfloat16
    assert A.select_blocks(_meta(3, 32, 128), bounds, 0, None, None, 5, block_size=16).shape == (3, 8, 5)
    q = A.kv_append(_meta(*POOL), 0, _meta(3, 8, 128), _meta(3, 8, 128), None, None, query=_meta(3, 32, 128))
    assert q.shape == (3, 32, 128)


@pytest.mark.parametrize("kw", [
    dict(query=_meta(3, 30, 128)), dict(query=_meta(3, 0, 128)), dict(query=_meta(3, 32, 64)), dict(query=_meta(32, 128)),
    dict(query=_meta(3, 32, 128, dtype=torch.float16)), dict(query=_meta(3, 32, 128, requires_grad=True)),
    dict(query=_meta(3, 128, 32).transpose(1, 2)), dict(pool=_meta(64, 2, 1, 8, 16, 128)),
    dict(pool=_meta(64, 2, 2, 8, 16, 128, dtype=torch.float64)), dict(pool=_meta(64, 2, 2, 8, 128, 16).transpose(4, 5)),
    dict(out=_meta(3, 32, 64)), dict(out=_meta(3, 1, 128).expand(3, 32, 128)),
])
def test_attention_checks_its_operands(kw):
    with pytest.raises(ValueError, match="paged_attention"):
        _call(**kw)


def test_gradients_are_refused_only_where_they_would_be_recorded():
    with torch.no_grad():
        _call(query=_meta(3, 32, 128, requires_grad=True))


def test_outputs_that_share_memory_are_refused():
    q = torch.zeros(3, 32, 128, dtype=torch.bfloat16)
    for out in (q, q.view(-1).as_strided(q.shape, q.stride())):
        with pytest.raises(ValueError, match="shares memory"):
            A._check_output(out, q, "out", "x", q)
    A._check_output(torch.zeros_like(q), q, "out", "x", q)
    with pytest.raises(ValueError, match="overlap"):
        A._check_output(torch.zeros(1, 1, 128, dtype=torch.bfloat16).expand(3, 32, 128), q, "out", "x")


def test_cpu_tensors_are_refused():
    pool = torch.zeros(POOL, dtype=torch.bfloat16)
    q = torch.zeros(3, 32, 128, dtype=torch.bfloat16)
    t, n = torch.zeros(3, 4, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        A.paged_attention(q, pool, 0, t, n)
    with pytest.raises(ValueError, match="CUDA"):
        A.kv_append(pool, 0, q[:, :8], q[:, :8], t, n)
    with pytest.raises(ValueError, match="CUDA"):
        A.key_bounds(pool, 0, t, n)


@pytest.mark.parametrize("kw", [
    dict(key=_meta(3, 4, 128)), dict(value=_meta(2, 8, 128)), dict(query=_meta(2, 32, 128)),
    dict(query=_meta(3, 9, 128)), dict(query_out=_meta(3, 32, 128)),
])
def test_append_checks_its_operands(kw):
    kw = {**dict(key=_meta(3, 8, 128), value=_meta(3, 8, 128)), **kw}
    with pytest.raises(ValueError, match="kv_append"):
        A.kv_append(_meta(*POOL), 0, kw.pop("key"), kw.pop("value"), None, None, **kw)


@pytest.mark.parametrize("kw", [dict(keep=0), dict(keep=3, first=2, last=2), dict(first=-1), dict(last=-1)])
def test_select_checks_its_numbers(kw):
    kw = {**dict(keep=4), **kw}
    with pytest.raises(ValueError, match="select_blocks"):
        A.select_blocks(_meta(3, 32, 128), _meta(64, 2, 8, 2, 128), 0, None, None, kw.pop("keep"), block_size=16, **kw)


def test_rope_table_is_worked_out_in_64_bits():
    t = A.rope_table(64, 131072, theta=500000.0, device="cpu")
    assert t.shape == (131072, 64) and t.dtype == torch.float32
    for p in (0, 1, 777, 131071):
        for i in (0, 1, 17, 31):
            a = p * 500000.0 ** (-2 * i / 64)
            # float32 rounds by half a step at most; cos and sin in 64 bits lose 2e-16 * the angle
            assert abs(t[p, i].item() - math.cos(a)) <= 2.0 ** -25 + 1e-9
            assert abs(t[p, 32 + i].item() - math.sin(a)) <= 2.0 ** -25 + 1e-9
    own = A.rope_table(4, 3, inv_freq=torch.tensor([1.0, 0.5]), device="cpu")
    assert own.shape == (3, 4)
    assert abs(own[2, 1].item() - math.cos(1.0)) < 1e-6 and abs(own[2, 3].item() - math.sin(1.0)) < 1e-6
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=4, inv_freq=torch.ones(3))):
        with pytest.raises(ValueError):
            A.rope_table(positions=4, device="cpu", **bad)
