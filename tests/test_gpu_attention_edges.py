"""The paged operators where calls go wrong or values leave the ordinary range:
batches with bad rows, scores far apart, agents on a matched prefix, captured
calls whose inputs move on."""

import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from agentkv_b200 import AgentKVPool, PoolConfig
from agentkv_b200 import _native as N
from agentkv_b200 import attention as A
from agentkv_b200 import kernels as K
from agentkv_b200.hf_cache import AgentKVCache

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


# ── attention: one score far above very many others ──────────────────────────
@pytest.mark.parametrize("gap", [0.0, 8.0, 10.0, 13.0, 15.0, 17.0, 17.5, 18.0, 20.0])
@pytest.mark.parametrize("dtype,G,D", [(F16, 4, 128), (F16, 9, 64), (F16, 4, 256), (F16, 2, 80), (F16, 1, 96), (BF16, 4, 128),
                                       (F32, 2, 64)])
def test_small_weights_count_beside_a_large_one(dtype, G, D, gap):
    """The first key scores `gap` above all the others and its value is 0, as
    a model's first token often has it: the output is the others' share.

    With w_j = e^(x_j - max), of which the two 16-bit numbers of a weight leave out
    2^-18 w_j + 2^-36 (bf16: no second part) and 32-bit scores and the hardware's exp2
    1e-5 w_j (as derived for the plain cases), |error| <= u |o| +
    (2e-5 sum w |v| + 2^-36 sum |v|) / sum w.  An output below the type's normal range
    is off by half its smallest step."""
    n, H, bs = 100_001, 2, 16
    g = _gen(int(gap * 10) + D)
    blocks = -(-n // bs)
    pool = torch.zeros((blocks, 1, 2, H, bs, D), dtype=dtype, device=DEV)
    pool[:, 0, 1] = (1 + 0.5 * _randn(g, blocks, H, bs, D, dtype=F32)).to(dtype)
    pool[0, 0, 1, :, 0] = 0
    q = _randn(g, 1, H * G, D, dtype=F32).sign().to(dtype)  # of +-1: all the heads' scores at one gap
    q = q.view(H, G, D)[:, :1].expand(H, G, D).reshape(1, H * G, D).contiguous()
    pool[0, 0, 0, :, 0] = (q.view(H, G, D)[:, 0].float() * (gap / D)).to(dtype)
    table = torch.arange(blocks, dtype=torch.int32, device=DEV)[None]
    out, lse = A.paged_attention(q, pool, 0, table, torch.tensor([n], dtype=torch.int32, device=DEV), scale=1.0,
                                 return_lse=True, check=True)
    k, v = (pool[:, 0, i].double().permute(1, 0, 2, 3).reshape(H, 1, -1, D)[:, :, :n] for i in range(2))
    x = q.view(H, G, 1, D).double() @ k.transpose(2, 3)
    w = torch.exp(x - x.amax(3, keepdim=True))
    total = w.sum(3, keepdim=True)
    want = (w @ v / total).view(1, H * G, D)
    u = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * u
    allowed = (2e-5 * (w @ v.abs()) + 2.0 ** -36 * v.abs().sum(2, keepdim=True)) / total
    err = (out.double() - want).abs()
    assert (err <= u * want.abs() + tiny + allowed.view(1, H * G, D)).all(), (err / want.abs()).max().item()
    assert ((lse.double() - torch.logsumexp(x, 3).view(1, -1)).abs() <= 1e-4).all()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_fp16_scores_that_rise_step_by_step(D):
    """Scores that rise by less than what makes the running maximum move, then by
    more, over a range far wider than fp16's: no weight passes the largest fp16 number."""
    n, H, G, bs = 4_000, 1, 8, 16
    g = _gen(D)
    blocks = -(-n // bs)
    pool = _randn(g, blocks, 1, 2, H, bs, D, dtype=F16)
    rise = torch.linspace(-60, 60, blocks * bs, device=DEV)
    for order in (rise, rise.flip(0), rise[torch.randperm(rise.numel(), generator=g, device=DEV)]):
        pool[:, 0, 0] = 0
        pool[:, 0, 0, 0, :, 0] = order.view(blocks, bs).to(F16)
        q = torch.zeros(1, G, D, dtype=F16, device=DEV)
        q[0, :, 0] = torch.tensor([1.0, 0.5, 0.25, 2.0, -1.0, -0.5, 4.0, 0.0])
        table = torch.arange(blocks, dtype=torch.int32, device=DEV)[None]
        out, lse = A.paged_attention(q, pool, 0, table, torch.tensor([n], dtype=torch.int32, device=DEV), scale=1.0,
                                     return_lse=True, check=True)
        k, v = (pool[:, 0, i, 0].double().reshape(-1, D)[:n] for i in range(2))
        x = q[0].double() @ k.T
        w = torch.softmax(x, 1)
        want = w @ v
        err = (out[0].double() - want).abs()
        # scores up to 240 in 32 bits, scaled to base 2 and taken off one another: off by 3 * 2^-24 * 347 = 6e-5
        # of the weight each, with the rest as above
        allowed = 2.0 ** -11 * want.abs() + 1e-4 * (w @ v.abs()) + 2.0 ** -25
        assert (err <= allowed).all(), (err - allowed).max().item()
        assert ((lse[0].double() - torch.logsumexp(x, 1)).abs() <= 1e-3).all()


# ── AgentKVCache.attend, captured ────────────────────────────────────────────
def _one_head_cache(total=64, bs=8):
    pool = AgentKVPool(config=PoolConfig(total_blocks=total, block_size=bs, num_layers=1, num_kv_heads=1, head_dim=16,
                                         dtype="float16", device="cuda"))
    return pool, AgentKVCache(pool, pool.create_root([]))


def _capture(call):
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        out = call()
    return graph, out


def test_a_captured_cache_attention_outlives_later_steps():
    """Eager call, capture of the same call, later steps with other lengths and
    more blocks, and memory asked for again in between: the replay still
    attends over the tokens of its capture."""
    pool, cache = _one_head_cache()
    g = _gen(6)
    k, v, q = (_randn(g, 1, 1, 5, 16, dtype=F16) for _ in range(3))
    cache.store(k, v, 0)
    want = cache.attend(q, 0).clone()
    graph, got = _capture(lambda: cache.attend(q, 0))
    taken = []
    for n in (1, 30, 1, 200):  # past the table's room
        x, y = (_randn(g, 1, 1, n, 16, dtype=F16) for _ in range(2))
        cache.store(x, y, 0)
        cache.attend(y, 0)
        torch.cuda.synchronize()
        for size in range(1, 65):  # what was let go is handed out again, with contents that are no length or block
            taken.append(torch.full((size,), 2 ** 30 + 7, dtype=torch.int32, device=DEV))
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want), n
    assert K.read_status(pool._allocator._status)[0] == 0


def test_a_captured_cache_attention_follows_a_copied_block():
    """The tokens' last block is shared by a fork and copied when the agent
    goes on: the replay reads the agent's own, whatever the fork's becomes."""
    pool, cache = _one_head_cache()
    g = _gen(7)
    k, v, q = (_randn(g, 1, 1, 5, 16, dtype=F16) for _ in range(3))
    cache.store(k, v, 0)
    want = cache.attend(q, 0).clone()
    graph, got = _capture(lambda: cache.attend(q, 0))
    old = pool.get_block_ids(cache.handle)
    child = cache.fork()
    cache.store(k[:, :, :1], v[:, :, :1], 0)
    assert pool.get_block_ids(cache.handle) != old == pool.get_block_ids(child.handle)
    pool._allocator._kv_data[old[0]] = math.nan
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_a_cache_refuses_to_store_while_capturing():
    pool, cache = _one_head_cache()
    k = torch.ones(1, 1, 5, 16, dtype=F16, device=DEV)
    with pytest.raises(RuntimeError, match="capturing"):
        _capture(lambda: (k + 1, cache.store(k, k, 0)))
    torch.cuda.synchronize()
    cache.store(k, k, 0)
    assert torch.equal(cache.attend(k, 0), k)


# ── append on views of one fused projection ──────────────────────────────────
@pytest.mark.parametrize("layout", ["heads", "thirds", "by head"])
def test_append_turns_a_fused_projection_in_place(layout):
    """query, key and value as views of one buffer and the rotated queries over
    the queries: as with memory of their own, and keys and values untouched."""
    H, D, bs, rows, T = 2, 64, 8, 3, 9
    g = _gen(12)
    if layout == "heads":
        packed = _randn(g, T, 4 * H, D, dtype=BF16)
        q, k, v = packed[:, :2 * H], packed[:, 2 * H:3 * H], packed[:, 3 * H:]
    elif layout == "thirds":
        packed = _randn(g, T, 3, H, D, dtype=BF16)
        q, k, v = packed.unbind(1)
    else:
        packed = _randn(g, T, H, 3 * D, dtype=BF16)
        q, k, v = packed.split(D, 2)
    pools = [torch.zeros((9, 1, 2, H, bs, D), dtype=BF16, device=DEV) for _ in range(2)]
    table = torch.arange(9, dtype=torch.int32, device=DEV).view(rows, 3)
    lengths = torch.tensor([11, 4, 20], dtype=torch.int32, device=DEV)
    kw = dict(starts=[0, 5, 6, 9], rope=A.rope_table(D, 32, device=DEV), check=True)
    want = A.kv_append(pools[0], 0, k.contiguous(), v.contiguous(), table, lengths, query=q.contiguous(), **kw)
    before = k.clone(), v.clone()
    got = A.kv_append(pools[1], 0, k, v, table, lengths, query=q, query_out=q, **kw)
    assert got is q and torch.equal(q, want) and torch.equal(pools[0], pools[1])
    assert torch.equal(k, before[0]) and torch.equal(v, before[1])


# ── first launches ───────────────────────────────────────────────────────────
_FIRST = '''
import torch
from agentkv_b200 import AgentKVPool, PoolConfig, attention as A
dev = torch.device("cuda", 0)
AgentKVPool(config=PoolConfig(total_blocks=4, block_size=16, num_layers=1, num_kv_heads=1, head_dim=64,
                              dtype="float16", device="cuda"))
forms = []
for dtype in (torch.float16, torch.bfloat16, torch.float32):
    for D, group in ((12, 1), (12, 4), (12, 5), (100, 2), (100, 3), (100, 8), (204, 1), (204, 4), (204, 7), (7, 1), (130, 9)):
        pool = torch.ones((3, 1, 2, 1, 16, D), dtype=dtype, device=dev)
        forms.append((torch.ones((1, group, D), dtype=dtype, device=dev), pool))
table = torch.tensor([[2, 0]], dtype=torch.int32, device=dev)
lengths = torch.tensor([20], dtype=torch.int32, device=dev)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, capture_error_mode="global"):
    outs = [A.paged_attention(q, pool, 0, table, lengths) for q, pool in forms]
graph.replay()
torch.cuda.synchronize()
assert all((o == 1).all() for o in outs)
print("right")
'''


def test_first_launches_of_every_form_inside_a_capture():
    """A pool's making loads the kernels: head dims and alignments of every
    form can be captured without an eager call of theirs before."""
    r = subprocess.run([sys.executable, "-c", _FIRST], capture_output=True, text=True, timeout=300,
                       cwd=Path(__file__).resolve().parents[1])
    assert r.returncode == 0 and "right" in r.stdout, r.stderr[-2000:]


# ── DecodeBatch: errors come back ────────────────────────────────────────────
def _batch(agents=2, bs=4, D=16, **kw):
    pool = AgentKVPool(config=PoolConfig(total_blocks=64, block_size=bs, num_layers=1, num_kv_heads=1, head_dim=D,
                                         dtype="float16", device="cuda"))
    handles = [pool.create_root([]) for _ in range(agents)]
    return pool, handles, pool.decode_batch(handles, **kw)


def test_a_rope_table_that_is_too_short_is_refused_on_the_host():
    pool, _, batch = _batch()
    x = torch.ones(2, 1, 16, dtype=F16, device=DEV)
    batch.advance([[1] * 6, [2]])
    k = torch.ones(7, 1, 16, dtype=F16, device=DEV)
    with pytest.raises(ValueError, match="rope table of 5 positions for 6 tokens"):
        batch.append(0, k, k, rope=A.rope_table(16, 5, device=DEV))
    batch.append(0, k, k, rope=A.rope_table(16, 6, device=DEV))
    batch.advance([[], [3]])  # the long row sits this one out: its positions are not turned
    batch.append(0, x[:1], x[:1], rope=A.rope_table(16, 5, device=DEV))
    batch.check()


def test_what_a_captured_step_reports_is_raised_by_a_later_advance():
    """A captured append whose rope table the rows outgrow: the next advances
    raise it, before anything changes, and the batch goes on once it is clear."""
    pool, (a, b), batch = _batch(width=4)
    x = torch.ones(2, 1, 16, dtype=F16, device=DEV)
    rope = A.rope_table(16, 3, device=DEV)
    batch.advance([[1], [2]])
    batch.append(0, x, x, rope=rope, check=True)
    graph, _ = _capture(lambda: batch.append(0, x, x, rope=rope))
    with pytest.raises(K.BlockOpError):
        for _ in range(6):
            batch.advance([[1], [2]])
            graph.replay()
            torch.cuda.synchronize()
    held = len(a.tokens)
    assert held in (4, 5) and len(b.tokens) == held
    batch.check()  # cleared
    batch.advance([[1], [2]])
    assert len(a.tokens) == held + 1
    batch.append(0, x, x)
    batch.check()
    graph.replay()
    with pytest.raises(K.BlockOpError):
        batch.check()
    batch.check()


def test_what_attend_reports_is_the_batch_s_own():
    """Not the allocator's record, behind which its own calls would stop."""
    pool, _, batch = _batch(bounds=True)
    x = torch.ones(2, 1, 16, dtype=F16, device=DEV)
    batch.advance([[1] * 9, [2] * 9])
    k = torch.ones(18, 1, 16, dtype=F16, device=DEV)
    batch.append(0, k, k)
    batch.check()
    batch.tables[0, 1] = 64
    batch.attend(0, x)
    with pytest.raises(K.BlockOpError):
        batch.check()
    batch.attend(0, x, keep=2)
    with pytest.raises(K.BlockOpError):
        batch.check()
    pool._allocator.check()
    batch.advance([[1], [2]])  # the tables are made anew
    batch.append(0, x, x)
    assert torch.equal(batch.attend(0, x, check=True), x)


# ── one block of more than 2^31 bytes per head ───────────────────────────────
def test_rows_beyond_32_bits_inside_a_block():
    """The earlier keys of a first block are read for its bounds, and a row is
    attended over, where a position's bytes start beyond 2^31 in its head's tile."""
    bs, D, n = 1 << 22, 256, 2_200_001
    pool = torch.zeros((1, 1, 2, 1, bs, D), device=DEV)  # 8.6 GB
    far = 2_150_000
    assert far * D * 4 > 2 ** 31
    g = _gen(1)
    kfar, vfar, k, v = (_randn(g, D, dtype=F32) for _ in range(4))
    pool[0, 0, 0, 0, far], pool[0, 0, 1, 0, far] = kfar, vfar
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    lengths = torch.tensor([n], dtype=torch.int32, device=DEV)
    bounds = torch.full((1, 1, 1, 2, D), 7.0, device=DEV)
    A.kv_append(pool, 0, k.view(1, 1, D), v.view(1, 1, D), table, lengths, bounds=bounds, check=True)
    assert torch.equal(pool[0, 0, 0, 0, n - 1], k) and torch.equal(pool[0, 0, 1, 0, n - 1], v)
    three = torch.stack([kfar, k, torch.zeros_like(k)])
    assert torch.equal(bounds[0, 0, 0, 0], three.amin(0)) and torch.equal(bounds[0, 0, 0, 1], three.amax(0))
    q = torch.zeros(1, 1, D, device=DEV)
    q[0, 0] = 30 * kfar / (kfar @ kfar)
    out = A.paged_attention(q, pool, 0, table, lengths, scale=1.0, check=True)
    x = torch.stack([q[0, 0].double() @ kfar.double(), q[0, 0].double() @ k.double()])
    w = torch.exp(x - 30)
    want = (w[0] * vfar.double() + w[1] * v.double()) / (w.sum() + (n - 2) * math.exp(-30))
    # scores of 30 in 32 bits, to base 2 and taken off one another: 3 * 2^-24 * 43 of a weight, with exp2's 2^-21
    assert ((out[0, 0].double() - want).abs() <= 2e-5 * (vfar.double().abs() + 1e-6)).all()


# ── lengths that are no lengths ──────────────────────────────────────────────
@pytest.mark.parametrize("wrong", [-1, -2 ** 31, 3 * 16 + 1, 2 ** 31 - 1])
def test_lengths_that_no_row_can_have_are_reported_by_every_operator(wrong):
    """And taken as 0, or as what the table holds, by those that read."""
    g = _gen(8)
    pool = _randn(g, 6, 1, 2, 2, 16, 64, dtype=BF16)
    table = torch.arange(6, dtype=torch.int32, device=DEV).view(2, 3)
    right = torch.tensor([20, 0 if wrong < 0 else 48], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([20, wrong], dtype=torch.int32, device=DEV)
    q = _randn(g, 2, 8, 64, dtype=BF16)
    bounds = A.key_bounds(pool, 0, table, right, check=True)
    sel = A.select_blocks(q, bounds, 0, table, right, 2, block_size=16, check=True)
    out = A.paged_attention(q, pool, 0, table, right, check=True)
    st = torch.zeros(8, dtype=torch.int32, device=DEV)

    def reported(row=1):
        code, index, bid = K.read_status(st)[:3]
        st.zero_()
        return (code, index, bid) == (N.AKV_ERR_OUT_OF_RANGE, row, wrong)

    assert torch.equal(A.paged_attention(q, pool, 0, table, lengths, status=st), out) and reported()
    assert torch.equal(A.select_blocks(q, bounds, 0, table, lengths, 2, block_size=16, status=st), sel) and reported()
    assert torch.equal(A.key_bounds(pool, 0, table, lengths, status=st), bounds) and reported()
    before = pool.clone()
    A.kv_append(pool, 0, q[:, :2], q[:, 2:4], table, lengths, status=st)
    assert K.read_status(st)[:2] == (N.AKV_ERR_OUT_OF_RANGE, 1)
    assert torch.equal(pool[table[1].long()], before[table[1].long()])


def test_a_captured_call_refuses_to_wait():
    """check=True while capturing: refused before anything is recorded, so that
    the capture goes on."""
    g = _gen(2)
    pool = _randn(g, 4, 1, 2, 2, 16, 64, dtype=BF16)
    table = torch.arange(4, dtype=torch.int32, device=DEV).view(2, 2)
    lengths = torch.tensor([20, 5], dtype=torch.int32, device=DEV)
    q = _randn(g, 2, 8, 64, dtype=BF16)
    bounds = A.key_bounds(pool, 0, table, lengths, check=True)
    want = A.paged_attention(q, pool, 0, table, lengths, check=True)

    def calls():
        for call in (lambda: A.paged_attention(q, pool, 0, table, lengths, check=True),
                     lambda: A.select_blocks(q, bounds, 0, table, lengths, 1, first=0, last=0, block_size=16, check=True),
                     lambda: A.key_bounds(pool, 0, table, lengths, bounds, check=True),
                     lambda: A.kv_append(pool, 0, q[:, :2], q[:, 2:4], table, lengths, check=True)):
            with pytest.raises(RuntimeError, match="capturing"):
                call()
        return A.paged_attention(q, pool, 0, table, lengths)

    graph, out = _capture(calls)
    before = pool.clone()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(pool, before)


# ── DecodeBatch over the shared tree ─────────────────────────────────────────
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_agents_on_a_matched_prefix_decode_together(dtype):
    """One agent commits its prompt's whole blocks; others match them (in whole,
    in part, by create_root), bring their own rest and go on, forks among them: outputs and
    bytes against a model that keeps each agent's keys and values apart."""
    H, G, D, L, bs = 2, 2, 64, 2, 8
    t = {"bfloat16": BF16, "float32": F32}[dtype]
    u = torch.finfo(t).eps / 2
    pool = AgentKVPool(config=PoolConfig(total_blocks=200, block_size=bs, num_layers=L, num_kv_heads=H, head_dim=D,
                                         dtype=dtype, device="cuda"))
    g = _gen(31)
    model = {}  # handle id -> [[keys, values] of each layer]

    def step(batch, new, **kw):
        batch.advance(new)
        counts = [len(n) for n in new]
        for layer in range(L):
            k, v = (_randn(g, sum(counts), H, D, dtype=t) for _ in range(2))
            batch.append(layer, k, v)
            at = 0
            for h, n in zip(batch.handles, counts):
                old = model[h.handle_id][layer]
                model[h.handle_id][layer] = [torch.cat([old[0], k[at:at + n]]), torch.cat([old[1], v[at:at + n]])]
                at += n
            q = _randn(g, batch.rows, H * G, D, dtype=t)
            out = batch.attend(layer, q, **kw)
            batch.check()
            data = pool._allocator._kv_data
            for i, h in enumerate(batch.handles):
                keys, values = model[h.handle_id][layer]
                ids = torch.tensor(pool.get_block_ids(h), device=DEV)
                held = data[ids, layer].permute(1, 2, 0, 3, 4).reshape(2, H, -1, D)[:, :, :len(h.tokens)]
                assert torch.equal(held[0].transpose(0, 1), keys) and torch.equal(held[1].transpose(0, 1), values)
                x = torch.einsum("hgd,nhd->hgn", q[i].view(H, G, D).double(), keys.double()) * D ** -0.5
                want = torch.einsum("hgn,nhd->hgd", torch.softmax(x, 2), values.double()).reshape(H * G, D)
                assert ((out[i].double() - want).abs() <= u * want.abs() + 3e-5 * 6).all()

    def empty(h):
        model[h.handle_id] = [[torch.zeros(0, H, D, dtype=t, device=DEV)] * 2 for _ in range(L)]
        return h

    def follow(h, of, n):
        model[h.handle_id] = [[x[:n] for x in layer] for layer in model[of.handle_id]]
        return h

    prompt = list(range(100, 137))  # 37 tokens: 4 blocks of 8 and 5 more
    a = empty(pool.create_root([]))
    first = pool.decode_batch([a], bounds=True)
    step(first, [prompt])
    pool.commit_prefix(a, 32)
    step(first, [[7]])                              # its own last block, behind the shared ones
    b, n = pool._tree.match_prefix(prompt + [1, 2])  # all that was committed
    assert n == 32
    follow(b, a, 32)
    c = pool.create_root(prompt[:32])                # the same, to the token
    follow(c, a, 32)
    d, n = pool._tree.match_prefix(prompt[:32] + [9] * 20)
    follow(d, a, 32)
    batch = pool.decode_batch([b, c, d, a], rows=5, bounds=first.bounds)
    step(batch, [prompt[32:] + [1, 2], [], [9] * 20, [8]])
    step(batch, [[3], [4], [5], [6]], keep=7)         # no row has more than 7 blocks: all of them
    pool.commit_prefix(d, 16)                         # deeper in the tree
    e, n = pool._tree.match_prefix(prompt[:32] + [9] * 20)
    assert n == 48
    follow(e, d, 48)
    f = pool.fork(e)
    follow(f, e, 48)
    for h in (b, c):
        pool.free(h)
    last = pool.decode_batch([d, e, f, a])
    for _ in range(bs + 1):
        step(last, [[1], [2], [3], [4]])
    pool._allocator.check()


def test_tokens_without_blocks_are_refused():
    """A root made of a prompt holds its tokens, but no key or value of those
    that no prefix matched."""
    pool, _, _ = _batch()
    h = pool.create_root(list(range(9)))
    with pytest.raises(ValueError, match="9 tokens in 0 blocks"):
        pool.decode_batch([h])
    pool.allocate_blocks(h, 3)  # for keys and values that come by other means
    batch = pool.decode_batch([h])
    pool.append_tokens(h, [1] * 4)
    with pytest.raises(ValueError, match="13 tokens in 3 blocks"):
        batch.advance([[1]])
    assert len(h.tokens) == 13 and len(pool.get_block_ids(h)) == 3


# ── infinite values ──────────────────────────────────────────────────────────
@pytest.mark.parametrize("dtype,D", [(F16, 64), (BF16, 128), (BF16, 80), (F32, 64), (BF16, 7)])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_a_value_that_is_no_number_stays_in_its_dimension(dtype, D, value):
    """Of its key head and row: infinite or NaN there, and all else as without it;
    behind the row's last position it is not there at all."""
    g = _gen(14)
    pool = _randn(g, 12, 1, 2, 2, 16, D, dtype=dtype)
    table = torch.arange(12, dtype=torch.int32, device=DEV).view(3, 4)
    lengths = torch.tensor([50, 60, 7], dtype=torch.int32, device=DEV)
    q = _randn(g, 3, 6, D, dtype=dtype)
    clean, lse = A.paged_attention(q, pool, 0, table, lengths, return_lse=True, check=True)
    pool[5, 0, 1, 1, 3, 2] = value   # row 1, position 19, key head 1, dimension 2
    pool[8, 0, 1, 1, 7:, 2] = value  # row 2, behind its 7 tokens
    pool[8, 0, 0, :, 7:] = value
    pool[3, 0, :, :, 2:] = value     # row 0, behind its 50
    out, l2 = A.paged_attention(q, pool, 0, table, lengths, return_lse=True, check=True)
    assert not torch.isfinite(out[1, 3:, 2]).any()
    out[1, 3:, 2] = clean[1, 3:, 2]
    assert torch.equal(out, clean) and torch.equal(l2, lse)
