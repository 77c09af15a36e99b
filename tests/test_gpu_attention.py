"""kv_append, paged_attention, select_blocks and key_bounds against their
definitions in 64 bits, and DecodeBatch / AgentKVCache.attend on them.

Tolerances, with u half a step of the type relative to the value
(finfo(t).eps / 2), derived before the first run:
* attention in 16 bits: the output is rounded once (u |o|).  Scores in 32 bits
  are off by at most 2^-22 of sum |q k| scale (256 products summed, each
  addition 2^-24 of the running sum, ~4 of them met on average by a chain of
  matrix products), here < 40 * 2^-22 = 1e-5; weights carry 2^-21 (the
  hardware's exp2) and, as two 16-bit numbers, u^2; together under 3e-5 of
  max |v|.  So |error| <= u |o| + 3e-5 max |v|, v ~ N(0, 1) below 6.
* attention in 32 bits: the same without the rounding of weights: 3e-5 max |v|.
* rotation: two products and a sum in 32 bits, the table rounded to 32 bits:
  4 * 2^-24 (|x| + |y|), then u of the result.
"""

import math

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


def _setup(dtype, H, D, bs, lengths, seed=0, layers=2, poison=True, extra=3):
    """A pool whose rows hold `lengths` tokens in shuffled blocks; everything
    that no row holds is NaN."""
    g = _gen(seed)
    need = [-(-n // bs) for n in lengths]
    total = sum(need) + extra
    perm = torch.randperm(total, generator=g, device=DEV).cpu()
    W = max(max(need, default=0), 1) + 1
    table = torch.full((len(lengths), W), 10 ** 6, dtype=torch.int32)  # behind a row: ids that must not be read
    pool = torch.full((total, layers, 2, H, bs, D), math.nan if poison else 0.0, dtype=dtype, device=DEV)
    at = 0
    for s, n in enumerate(lengths):
        ids = perm[at:at + need[s]]
        table[s, :need[s]] = ids.int()
        at += need[s]
        for j, b in enumerate(ids.tolist()):
            k = min(bs, n - j * bs)
            pool[b, :, :, :, :k] = _randn(g, layers, 2, H, k, D, dtype=dtype)
    return pool, table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), g


def _kv(pool, table, s, n, layer):
    bs = pool.shape[4]
    ids = table[s, :-(-n // bs)].long()
    d = pool[ids, layer].double()  # [blocks, 2, H, bs, D]
    return d.permute(1, 2, 0, 3, 4).reshape(2, pool.shape[3], -1, pool.shape[5])[:, :, :n]


def _want(query, pool, table, lengths, layer, scale, window=0, selected=None):
    S, Hq, D = query.shape
    H, bs = pool.shape[3], pool.shape[4]
    G = Hq // H
    out = torch.zeros(S, Hq, D, dtype=torch.float64, device=DEV)
    lse = torch.full((S, Hq), -math.inf, dtype=torch.float64, device=DEV)
    for s, n in enumerate(lengths.tolist()):
        if n <= 0:
            continue
        k, v = _kv(pool, table, s, n, layer)
        for h in range(H):
            pos = torch.arange(n, device=DEV)
            held = pos >= n - window if window else torch.ones(n, dtype=torch.bool, device=DEV)
            if selected is not None:
                sel = selected[s, h][selected[s, h] >= 0].long()
                held &= torch.isin(pos // bs, sel)
            if not held.any():
                continue
            x = query[s, h * G:(h + 1) * G].double() @ k[h][held].T * scale
            lse[s, h * G:(h + 1) * G] = torch.logsumexp(x, 1)
            out[s, h * G:(h + 1) * G] = torch.softmax(x, 1) @ v[h][held]
    return out, lse


def _check(out, want, dtype):
    u = torch.finfo(dtype).eps / 2 if dtype != F32 else 2.0 ** -24
    err = (out.double() - want).abs()
    assert torch.isfinite(out).all()
    assert (err <= u * want.abs() + 3e-5 * 6).all(), (err - u * want.abs()).max().item()


def _attend(query, pool, table, lengths, layer, **kw):
    st = torch.zeros(8, dtype=torch.int32, device=DEV)
    out = A.paged_attention(query, pool, layer, table, lengths, status=st, **kw)
    assert K.read_status(st)[0] == 0
    return out


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("H,G,D,bs", [(2, 4, 128, 16), (1, 1, 64, 16), (3, 8, 64, 8), (2, 9, 128, 32), (1, 20, 96, 64),
                                      (2, 3, 256, 16), (2, 2, 80, 16), (1, 5, 12, 4), (2, 7, 7, 1), (1, 16, 256, 8),
                                      (8, 4, 128, 128), (2, 2, 128, 2), (1, 3, 100, 16)])
def test_lengths_from_none_to_many_chunks(dtype, H, G, D, bs):
    lengths = [1, 0, 2, 15, 16, 17, 63, 64, 65, 0, 129, 500]
    pool, table, lens, g = _setup(dtype, H, D, bs, lengths, seed=D)
    q = _randn(g, len(lengths), H * G, D, dtype=dtype)
    for layer in (0, 1):
        out, lse = _attend(q, pool, table, lens, layer, return_lse=True)
        want, wl = _want(q, pool, table, lens, layer, D ** -0.5)
        _check(out, want, dtype)
        assert torch.equal(lse.isinf(), wl.isinf()) and (lse < 0)[lse.isinf()].all()
        fin = ~wl.isinf()
        assert ((lse.double() - wl)[fin].abs() <= 1e-4).all()


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F32, 64)])
def test_one_long_row_over_every_cta(dtype, D):
    pool, table, lens, g = _setup(dtype, 1, D, 16, [70001, 3], layers=1)
    q = _randn(g, 2, 4, D, dtype=dtype)
    out = _attend(q, pool, table, lens, 0, scale=0.3)
    _check(out, _want(q, pool, table, lens, 0, 0.3)[0], dtype)


def test_many_rows_more_than_threads():
    lengths = [(i * 37) % 90 for i in range(700)]
    pool, table, lens, g = _setup(BF16, 2, 64, 16, lengths, layers=1)
    q = _randn(g, 700, 4, 64, dtype=BF16)
    _check(_attend(q, pool, table, lens, 0), _want(q, pool, table, lens, 0, 0.125)[0], BF16)


@pytest.mark.parametrize("dtype,D,bs", [(BF16, 128, 16), (F16, 64, 4), (F32, 96, 32)])
@pytest.mark.parametrize("window", [1, 7, 64, 100, 10 ** 9])
def test_window_reads_nothing_before_it(dtype, D, bs, window):
    lengths = [1, 5, 64, 65, 300, 0, 511]
    pool, table, lens, g = _setup(dtype, 2, D, bs, lengths, seed=window % 97)
    for s, n in enumerate(lengths):  # blocks wholly before the window: freed
        table[s, :max(0, n - window) // bs] = 10 ** 6
    q = _randn(g, len(lengths), 6, D, dtype=dtype)
    out = _attend(q, pool, table, lens, 1, window=window)
    safe = table.clone()
    safe[safe == 10 ** 6] = 0
    pool0 = torch.where(pool.isnan(), torch.zeros_like(pool), pool)
    _check(out, _want(q, pool0, safe, lens, 1, D ** -0.5, window=window)[0], dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_selected_blocks(dtype):
    bs, H, G, D = 16, 2, 4, 128
    lengths = [1, 40, 0, 333, 1000]
    pool, table, lens, g = _setup(dtype, H, D, bs, lengths)
    keep = 9
    sel = torch.full((5, H, keep), -1, dtype=torch.int32)
    for s, n in enumerate(lengths):
        blocks = -(-n // bs)
        for h in range(H):
            pick = torch.randperm(blocks)[:max(0, min(keep - h, blocks))]  # any order, one entry fewer for head 1
            sel[s, h, :len(pick)] = pick.int()
    sel[4, 1] = -1  # nothing at all
    sel = sel.to(DEV)
    q = _randn(g, 5, H * G, D, dtype=dtype)
    out = _attend(q, pool, table, lens, 0, selected=sel)
    want, _ = _want(q, pool, table, lens, 0, D ** -0.5, selected=sel)
    assert (out[4, G:] == 0).all() and (out[2] == 0).all()
    _check(out, want, dtype)


def test_scale_of_any_sign_and_none():
    pool, table, lens, g = _setup(BF16, 2, 128, 16, [200, 65])
    q = _randn(g, 2, 8, 128, dtype=BF16)
    for scale in (0.0, -0.2, 1.0):
        _check(_attend(q, pool, table, lens, 0, scale=scale), _want(q, pool, table, lens, 0, scale)[0], BF16)


def test_infinities_and_nan_stay_with_their_row():
    """A row whose keys or values hold inf or NaN gives what softmax gives, and
    its neighbours' results are as without it."""
    pool, table, lens, g = _setup(F16, 2, 64, 16, [50, 50, 50, 50], layers=1)
    q = _randn(g, 4, 8, 64, dtype=F16)
    clean = _attend(q, pool, table, lens, 0)
    pool[table[1, 1].long(), 0, 1, :, 3] = math.nan   # a value
    pool[table[2, 2].long(), 0, 0, :, 0] = math.inf   # a key
    out = _attend(q, pool, table, lens, 0)
    assert torch.equal(out[[0, 3]], clean[[0, 3]])
    assert out[1].isnan().all()
    assert not torch.equal(out[2], clean[2])


def test_strided_queries_and_outputs():
    pool, table, lens, g = _setup(BF16, 2, 128, 16, [100, 37, 64])
    big = _randn(g, 3, 3, 8, 128, dtype=BF16)
    q = big[:, 1]                                     # rows 3 * 8 * 128 apart
    ref = _attend(q.contiguous(), pool, table, lens, 0)
    assert torch.equal(_attend(q, pool, table, lens, 0), ref)
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(_attend(heads_first, pool, table, lens, 0), ref)
    odd = torch.empty(3 * 8 * 128 + 1, dtype=BF16, device=DEV)[1:].view(3, 8, 128).copy_(q)  # 2-byte aligned
    _check(_attend(odd, pool, table, lens, 0), _want(q, pool, table, lens, 0, 128 ** -0.5)[0], BF16)
    room = torch.full((3, 16, 128), 7.0, dtype=BF16, device=DEV)
    out = room[:, ::2]
    _attend(q, pool, table, lens, 0, out=out)
    assert torch.equal(out, ref) and (room[:, 1::2] == 7).all()
    wide = torch.zeros(3, table.shape[1] + 5, dtype=torch.int32, device=DEV)
    wide[:, 5:] = table
    assert torch.equal(_attend(q, pool, wide[:, 5:], lens, 0), ref)
    expanded = _attend(q, pool, table[:1].expand(3, -1), lens.clamp(max=100), 0)
    assert torch.equal(expanded[0], ref[0])


def test_offsets_beyond_32_bits():
    """Blocks whose bytes start beyond 2^32."""
    H, bs, D = 8, 16, 128
    pool = torch.empty((70000, 1, 2, H, bs, D), dtype=BF16, device=DEV)  # 4.6 GB
    g = _gen(4)
    ids = torch.tensor([69999, 5, 66000, 40000], device=DEV)
    pool[ids] = _randn(g, 4, 1, 2, H, bs, D, dtype=BF16)
    table, lens = ids.int()[None], torch.tensor([61], dtype=torch.int32, device=DEV)
    q = _randn(g, 1, 32, D, dtype=BF16)
    _check(_attend(q, pool, table, lens, 0), _want(q, pool, table, lens, 0, D ** -0.5)[0], BF16)
    k = _randn(g, 1, H, D, dtype=BF16)
    A.kv_append(pool, 0, k, k, table, lens, check=True)
    assert torch.equal(pool[40000, 0, 0, :, 12], k[0]) and torch.equal(pool[40000, 0, 1, :, 12], k[0])


def test_bad_ids_and_lengths_are_reported_and_left_out():
    pool, table, lens, g = _setup(BF16, 2, 128, 16, [40, 40, 40], extra=0)
    q = _randn(g, 3, 8, 128, dtype=BF16)
    good = _attend(q, pool, table, lens, 0)
    bad = table.clone()
    bad[1, 1] = pool.shape[0]
    st = torch.zeros(8, dtype=torch.int32, device=DEV)
    out = A.paged_attention(q, pool, 0, bad, lens, status=st)
    assert K.read_status(st)[:3] == (N.AKV_ERR_OUT_OF_RANGE, 1, pool.shape[0])
    assert torch.equal(out[[0, 2]], good[[0, 2]]) and torch.isfinite(out).all()
    with pytest.raises(K.BlockOpError):
        A.paged_attention(q, pool, 0, bad, lens, status=st, check=True)
    bad[1, 1] = -5
    with pytest.raises(K.BlockOpError):
        A.paged_attention(q, pool, 0, bad, lens, check=True)
    long = lens.clone()
    long[2] = table.shape[1] * 16 + 1
    table2 = table.clone()
    table2[2, 3] = table2[2, 0]
    st.zero_()
    out = A.paged_attention(q, pool, 0, table2, long, status=st)
    assert K.read_status(st)[:2] == (N.AKV_ERR_OUT_OF_RANGE, 2)
    sel = torch.tensor([[[0, 7, -1]] * 2] * 3, dtype=torch.int32, device=DEV)
    st.zero_()
    A.paged_attention(q, pool, 0, table, lens, selected=sel, status=st)
    assert K.read_status(st)[0] == N.AKV_ERR_OUT_OF_RANGE
    assert torch.equal(_attend(q, pool, table, lens, 0), good)  # and the next call is whole again


def test_nothing_to_do():
    """No rows, tables of no width, batches of padding alone."""
    pool = torch.zeros((4, 1, 2, 2, 16, 64), dtype=BF16, device=DEV)
    bounds = torch.zeros((4, 1, 2, 2, 64), dtype=BF16, device=DEV)
    for rows, width in ((0, 3), (3, 0), (3, 2)):
        q = torch.ones(rows, 4, 64, dtype=BF16, device=DEV)
        t = torch.zeros(rows, width, dtype=torch.int32, device=DEV)
        n = torch.zeros(rows, dtype=torch.int32, device=DEV)
        out, lse = A.paged_attention(q, pool, 0, t, n, return_lse=True, check=True)
        assert out.shape == q.shape and (out == 0).all() and (lse == -math.inf).all()
        sel = A.select_blocks(q, bounds, 0, t, n, 3, block_size=16, check=True)
        assert sel.shape == (rows, 2, 3) and (sel == -1).all()
        k = q[:, :2]
        if rows:  # the queries' result over the keys
            with pytest.raises(ValueError, match="query_out shares memory"):
                A.kv_append(pool, 0, k, k, t, n, query=q, query_out=q, check=True)
            k = k.clone()
        assert torch.equal(A.kv_append(pool, 0, k, k, t, n, query=q, query_out=q, check=True), q)
        A.key_bounds(pool, 0, t, n, bounds, check=True)
        assert (pool == 0).all() and (bounds == 0).all()


def test_reads_go_on_behind_an_error():
    pool, table, lens, g = _setup(BF16, 2, 64, 16, [40, 700], layers=1)
    bounds = A.key_bounds(pool, 0, table, lens)
    q = _randn(g, 2, 8, 64, dtype=BF16)
    sel = A.select_blocks(q, bounds, 0, table, lens, 5, block_size=16)
    out = _attend(q, pool, table, lens, 0, selected=sel)
    st = torch.zeros(8, dtype=torch.int32, device=DEV)
    st[0] = N.AKV_ERR_OUT_OF_RANGE
    assert torch.equal(A.select_blocks(q, bounds, 0, table, lens, 5, block_size=16, status=st), sel)
    assert torch.equal(A.paged_attention(q, pool, 0, table, lens, selected=sel, status=st), out)
    before = pool.clone()
    A.kv_append(pool, 0, q[:, :2], q[:, :2], table, lens, status=st)
    assert torch.equal(pool.nan_to_num(3.0), before.nan_to_num(3.0))


# ── append ───────────────────────────────────────────────────────────────────
def _rotate64(x, pos, rot, interleaved, theta=10000.0):
    x = x.double().clone()
    inv = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    a = pos.double()[:, None, None] * inv
    i = torch.arange(0, rot, 2, device=DEV) if interleaved else torch.arange(rot // 2, device=DEV)
    j = i + (1 if interleaved else rot // 2)
    u, v = x[..., i].clone(), x[..., j].clone()
    x[..., i], x[..., j] = u * a.cos() - v * a.sin(), v * a.cos() + u * a.sin()
    return x


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("H,G,D,bs,rot,inter", [(2, 4, 128, 16, 128, False), (2, 3, 64, 8, 64, True), (1, 1, 80, 16, 32, False),
                                                (3, 2, 96, 4, 48, True), (2, 5, 256, 32, 128, False), (1, 2, 12, 4, 6, False),
                                                (2, 1, 7, 2, 6, True), (1, 2, 7, 1, 2, False), (2, 2, 128, 64, 0, False)])
@pytest.mark.parametrize("ragged", [False, True])
def test_append(dtype, H, G, D, bs, rot, inter, ragged):
    old = [0, 5, 15, 16, 40, 0, 63, 7]
    new = [1, 3, 1, 17, 0, 70, 2, 1] if ragged else [1] * 8
    lens = [o + n for o, n in zip(old, new)]
    if not ragged:
        lens[4], new[4] = 0, 0  # a padding row
    pool, table, lengths, g = _setup(dtype, H, D, bs, lens, seed=D + bs)
    pool = torch.where(pool.isnan(), torch.zeros_like(pool), pool)
    T = sum(new) + 2 if ragged else 8
    k, v, q = (_randn(g, T, n, D, dtype=dtype) for n in (H, H, H * G))
    rope = A.rope_table(rot, 200, device=DEV) if rot else None
    starts = None
    if ragged:
        s = [0]
        for n in new:
            s.append(s[-1] + n)
        starts = torch.tensor(s, dtype=torch.int32, device=DEV)
    bounds = torch.full((pool.shape[0], 2, H, 2, D), 5.0, dtype=dtype, device=DEV)
    before, b0 = pool.clone(), bounds.clone()
    qo = torch.full_like(q, 3.0)
    kw = dict(starts=starts, rope=rope, interleaved=inter, query=q, query_out=qo, bounds=bounds, check=True)
    got = A.kv_append(pool, 1, k, v, table, lengths, **kw)
    assert got is qo
    u = torch.finfo(dtype).eps / 2 if dtype != F32 else 2.0 ** -24
    want_pool, used = before.clone(), torch.zeros(pool.shape[0], dtype=torch.bool)
    row_used = torch.zeros(T, dtype=torch.bool)
    for s, (n, length) in enumerate(zip(new, lens)):
        r0 = int(starts[s]) if ragged else s
        for i in range(n):
            p = length - n + i
            b = int(table[s, p // bs])
            pos = torch.tensor([p], device=DEV)
            r = r0 + i
            row_used[r] = True
            for x, y in ((k[r:r + 1], pool[b, 1, 0, :, p % bs][None]), (q[r:r + 1], qo[r:r + 1])):
                w = _rotate64(x, pos, rot, inter) if rot else x.double()
                mag = x.double().abs()
                mag = mag if not rot else mag + mag.amax(-1, keepdim=True)
                assert ((y.double() - w).abs() <= u * w.abs() + 4 * 2.0 ** -24 * mag).all()
            assert torch.equal(pool[b, 1, 1, :, p % bs], v[r])
            want_pool[b, 1, :, :, p % bs] = pool[b, 1, :, :, p % bs]
            used[b] = True
            held = pool[b, 1, 0, :, :min(bs, length - p // bs * bs)]
            assert torch.equal(bounds[b, 1, :, 0], held.amin(1)) and torch.equal(bounds[b, 1, :, 1], held.amax(1))
    assert torch.equal(pool, want_pool)  # nothing else moved
    b0[used, 1] = bounds[used, 1]
    assert torch.equal(bounds, b0)
    assert (qo[~row_used] == 3).all()  # padding rows are left
    again = pool.clone()
    A.kv_append(pool, 1, k, v, table, lengths, **{**kw, "query_out": q, "query": q})  # in place, and the same again
    assert torch.equal(pool, again) and torch.equal(q[row_used], qo[row_used])


def test_append_from_strided_states_and_nan_bounds():
    H, D, bs = 2, 64, 16
    pool, table, lengths, g = _setup(BF16, H, D, bs, [20, 33], poison=False)
    hf = _randn(g, 1, H, 2, D, dtype=BF16)  # [1, heads, tokens, head_dim]
    kv = _randn(g, 2, 3 * H, D, dtype=BF16)
    bounds = torch.zeros((pool.shape[0], 2, H, 2, D), dtype=BF16, device=DEV)
    hf[0, 1, 1, 5] = math.nan
    A.kv_append(pool, 0, hf[0].transpose(0, 1), kv[:, H:2 * H], table, lengths, bounds=bounds, check=True)
    for s, n in enumerate([20, 33]):
        b = int(table[s, (n - 1) // bs])
        assert torch.equal(pool[b, 0, 0, :, (n - 1) % bs].nan_to_num(9.0), hf[0, :, s].nan_to_num(9.0))
        assert torch.equal(pool[b, 0, 1, :, (n - 1) % bs], kv[s, H:2 * H])
    b = int(table[1, 2])
    assert bounds[b, 0, 1, :, 5].isnan().all() and torch.isfinite(bounds[b, 0, 0]).all()


def test_append_refuses_on_the_device():
    pool, table, lengths, g = _setup(F16, 2, 64, 16, [20, 33, 5], poison=False)
    k = _randn(g, 3, 2, 64, dtype=F16)
    rope = A.rope_table(64, 30, device=DEV)
    before = pool.clone()
    st = torch.zeros(8, dtype=torch.int32, device=DEV)
    A.kv_append(pool, 0, k, k, table, lengths, rope=rope, status=st)
    assert K.read_status(st)[:3] == (N.AKV_ERR_OUT_OF_RANGE, 1, 32)  # position 32 of 30
    A.kv_append(pool, 0, k, k, table, lengths, status=st)            # the error sticks: nothing happens
    b = int(table[1, 2])
    assert torch.equal(pool[b], before[b])
    with pytest.raises(K.BlockOpError):
        K.raise_for_status(st)
    bad = table.clone()
    bad[0, 1] = -1
    A.kv_append(pool, 0, k, k, bad, lengths, status=st)
    assert K.read_status(st)[:3] == (N.AKV_ERR_OUT_OF_RANGE, 0, -1)
    for starts in ([0, 1, 9, 10], [0, 2, 1, 3], [-1, 1, 2, 3], [0, 25, 26, 27]):
        st.zero_()
        A.kv_append(pool, 0, k, k, table, lengths, starts=torch.tensor(starts, dtype=torch.int32, device=DEV), status=st)
        assert K.read_status(st)[0] == N.AKV_ERR_OUT_OF_RANGE, starts
    with pytest.raises(ValueError, match="16-byte"):
        A.kv_append(pool, 0, k, k, table, lengths, rope=torch.zeros(32 * 64 + 1, device=DEV)[1:].view(32, 64))


# ── selection ────────────────────────────────────────────────────────────────
def _want_blocks(q, bounds, table, lengths, layer, bs, keep, first, last):
    S, H = q.shape[0], bounds.shape[2]
    G = q.shape[1] // H
    out = torch.full((S, H, keep), -1, dtype=torch.int32)
    for s, n in enumerate(lengths.tolist()):
        blocks = -(-max(n, 0) // bs)
        if blocks <= keep:
            out[s, :, :blocks] = torch.arange(blocks, dtype=torch.int32)
            continue
        box = bounds[table[s, :blocks].long(), layer].double()
        for h in range(H):
            x = q[s, h * G:(h + 1) * G].double()
            up, down = x.clamp(min=0).sum(0), x.clamp(max=0).sum(0)
            score = (box[:, h, 1] * up + box[:, h, 0] * down).sum(1)
            score = torch.where(score.isnan(), 1.8e308, score).clamp(-1.7976931348623157e308, 1.7976931348623157e308).tolist()
            always = [j for j in range(blocks) if j < first or j >= blocks - last]
            rest = sorted((j for j in range(first, blocks - last)), key=lambda j: (-score[j], j))
            out[s, h] = torch.tensor(sorted(always + rest[:keep - len(always)]), dtype=torch.int32)
    return out


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("H,G,D,keep,first,last", [(2, 4, 128, 8, 1, 1), (1, 1, 64, 1, 0, 0), (3, 2, 96, 12, 2, 3),
                                                   (1, 8, 256, 30, 0, 1), (2, 3, 12, 5, 0, 0), (1, 2, 7, 4, 4, 0),
                                                   (2, 1, 80, 6, 3, 3)])
def test_selection_is_the_one_in_64_bits(dtype, H, G, D, keep, first, last):
    bs = 16
    lengths = [0, 1, keep * bs, keep * bs + 1, 700, 1100, 333]
    pool, table, lens, g = _setup(dtype, H, D, bs, lengths, seed=keep)
    bounds = A.key_bounds(pool, 1, table, lens, check=True)
    for s, n in enumerate(lengths):  # the bounds themselves
        for j in range(-(-n // bs)):
            b = int(table[s, j])
            held = pool[b, 1, 0, :, :min(bs, n - j * bs)]
            assert torch.equal(bounds[b, 1, :, 0], held.amin(1)) and torch.equal(bounds[b, 1, :, 1], held.amax(1))
    q = _randn(g, len(lengths), H * G, D, dtype=dtype)
    got = A.select_blocks(q, bounds, 1, table, lens, keep, block_size=bs, first=first, last=last, check=True)
    assert torch.equal(got.cpu(), _want_blocks(q, bounds, table, lens, 1, bs, keep, first, last))


def _bounds_batch(n_blocks, H, D, dtype, seed):
    g = _gen(seed)
    b = _randn(g, n_blocks, 1, H, 2, D, dtype=dtype)
    b = torch.stack([b.amin(3), b.amax(3)], 3)
    table = torch.arange(n_blocks, dtype=torch.int32, device=DEV)[None]
    return b, table, torch.tensor([n_blocks * 16], dtype=torch.int32, device=DEV), g


@pytest.mark.parametrize("kind", ["alike", "two kinds", "last place", "nan", "inf", "zero query", "huge"])
def test_selection_at_the_border(kind):
    """Blocks that are equal, or differ in the last place of a long sum, or
    whose score is no number: the lowest places of equal scores are taken."""
    n, H, G, D = 600, 2, 4, 128
    b, table, lens, g = _bounds_batch(n, H, D, BF16, 5)
    q = _randn(g, 1, H * G, D, dtype=BF16)
    if kind == "alike":
        b[:] = b[:1].clone()
    elif kind == "two kinds":
        b[::2], b[1::2] = b[:1].clone(), b[1:2].clone()
    elif kind == "last place":  # one bound of each block apart from the first's by one step of the type
        b[:] = b[:1].clone()
        flat = b.view(torch.int16)
        pick = torch.randint(0, D, (n,), generator=g, device=DEV)
        flat[torch.arange(n, device=DEV), 0, :, 1, pick] += 1
    elif kind == "nan":
        b[100:140, :, 0, 1, 3] = math.nan
    elif kind == "inf":
        b[200:230, :, :, 1, 7] = math.inf
        b[300:310, :, :, 0, 9] = -math.inf
        b[7, :, :, :, 0] = -math.inf
    elif kind == "zero query":
        q.zero_()
    else:
        b *= 1e30
        q *= 1e9
    for keep in (1, 37, 300, 599):
        got = A.select_blocks(q, b, 0, table, lens, keep, block_size=16, first=0, last=0, check=True)
        assert torch.equal(got.cpu(), _want_blocks(q, b, table, lens, 0, 16, keep, 0, 0)), keep


@pytest.mark.parametrize("n", [8191, 8192, 8193, 20000])
def test_selection_over_long_tables(n):
    b, table, lens, g = _bounds_batch(n, 1, 64, F16, n)
    q = _randn(g, 1, 4, 64, dtype=F16)
    got = A.select_blocks(q, b, 0, table, lens, 500, block_size=16, first=1, last=2, check=True)
    assert torch.equal(got.cpu(), _want_blocks(q, b, table, lens, 0, 16, 500, 1, 2))


def test_selection_reports_bad_ids():
    b, table, lens, g = _bounds_batch(50, 1, 64, F16, 1)
    q = _randn(g, 1, 4, 64, dtype=F16)
    table[0, 17] = 50
    with pytest.raises(K.BlockOpError):
        A.select_blocks(q, b, 0, table, lens, 5, block_size=16, check=True)
    A.select_blocks(q, b, 0, table.clamp(max=49), lens, 5, block_size=16, check=True)


# ── streams and graphs ───────────────────────────────────────────────────────
def test_calls_on_two_streams_at_once():
    pool, table, lens, g = _setup(BF16, 2, 128, 16, [3000, 17, 900], layers=1)
    qs = [_randn(g, 3, 8, 128, dtype=BF16) for _ in range(2)]
    want = [_attend(q, pool, table, lens, 0) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(A.paged_attention(qs[i], pool, 0, table, lens))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


def test_two_captured_graphs_replayed_at_once_and_with_other_lengths():
    pool, table, lens, g = _setup(BF16, 2, 128, 16, [3000, 17, 900], layers=1)
    q = _randn(g, 3, 8, 128, dtype=BF16)
    bounds = A.key_bounds(pool, 0, table, lens)
    _attend(q, pool, table, lens, 0)
    graphs, outs, lengths = [], [], []
    for _ in range(2):
        n = lens.clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, capture_error_mode="thread_local"):
            full = A.paged_attention(q, pool, 0, table, n)
            sel = A.select_blocks(q, bounds, 0, table, n, 12, block_size=16)
            part = A.paged_attention(q, pool, 0, table, n, selected=sel)
        graphs.append(graph)
        outs.append((full, sel, part))
        lengths.append(n)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn, now in enumerate(([3000, 17, 900], [64, 0, 899], [1, 1, 1])):
        for n in lengths:
            n.copy_(torch.tensor(now, dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(5):
            for graph, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        n = torch.tensor(now, dtype=torch.int32, device=DEV)
        sel = A.select_blocks(q, bounds, 0, table, n, 12, block_size=16)
        want = (_attend(q, pool, table, n, 0), sel, _attend(q, pool, table, n, 0, selected=sel))
        for got in outs:
            assert all(torch.equal(a, b) for a, b in zip(got, want)), turn


# ── together ─────────────────────────────────────────────────────────────────


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_agents_decode_together(dtype):
    """A prompt appended in one step, forked agents that share its last, partly
    filled block, uneven steps of them through append, dense, windowed and sparse attention: every output and
    the pool's bytes against a model that keeps each agent's keys and values apart."""
    H, G, D, L, bs = 2, 3, 64, 2, 16
    t = {"bfloat16": BF16, "float32": F32}[dtype]
    pool = AgentKVPool(config=PoolConfig(total_blocks=160, block_size=bs, num_layers=L, num_kv_heads=H, head_dim=D,
                                         dtype=dtype, device="cuda"))
    g = _gen(2)
    rope = A.rope_table(D, 400, device=DEV)
    model = {}  # agent -> per layer ([n, H, D] rotated keys, values) in 64 bits, as rounded

    def step(batch, names, counts):
        T = sum(counts)
        rows = len(names)
        batch.advance([[7] * n for n in counts])
        for layer in range(L):
            k, v = _randn(g, T, H, D, dtype=t), _randn(g, T, H, D, dtype=t)
            batch.append(layer, k, v, rope=rope, check=True)
            at = 0
            for name, n in zip(names, counts):
                old = model[name][layer]
                pos = torch.arange(old[0].shape[0], old[0].shape[0] + n, device=DEV)
                kr = _rotate64(k[at:at + n], pos, D, False).to(t).double()
                model[name][layer] = (torch.cat([old[0], kr]), torch.cat([old[1], v[at:at + n].double()]))
                at += n
            q = _randn(g, batch.rows, H * G, D, dtype=t)
            for kw in (dict(), dict(window=20), dict(keep=4, first=1, last=2)):
                out = batch.attend(layer, q, check=True, **kw)
                assert (out[rows:] == 0).all()
                sel = A.select_blocks(q, batch.bounds, layer, batch.tables, batch.lengths, 4, block_size=bs, first=1,
                                      last=2) if "keep" in kw else None
                for i, name in enumerate(names):
                    ks, vs = model[name][layer]
                    n = ks.shape[0]
                    p = torch.arange(n, device=DEV)
                    for h in range(H):
                        held = p >= n - kw.get("window", n)
                        if sel is not None:
                            held = torch.isin(p // bs, sel[i, h].long())
                        x = q[i, h * G:(h + 1) * G].double() @ ks[held, h].T * D ** -0.5
                        # keys may differ from the model's in the last place: two roundings of near-ties
                        want = torch.softmax(x, 1) @ vs[held, h]
                        u = torch.finfo(t).eps / 2
                        err = (out[i, h * G:(h + 1) * G].double() - want).abs()
                        assert (err <= u * want.abs() + 3e-5 * 6 + u * 6).all()

    root = pool.create_root([])
    model["root"] = [(torch.zeros(0, H, D, dtype=torch.float64, device=DEV),) * 2 for _ in range(L)]
    first = pool.decode_batch([root], bounds=True)
    step(first, ["root"], [70])
    kids = pool.fork_many(root, 5)
    names = [f"k{i}" for i in range(5)]
    for n in names:
        model[n] = [tuple(x.clone() for x in m) for m in model["root"]]
    batch = pool.decode_batch(kids, rows=7, bounds=first.bounds)
    step(batch, names, [1] * 5)
    step(batch, names, [3, 0, 17, 1, 1])
    for _ in range(2):
        step(batch, names, [1] * 5)
    step(first, ["root"], [1])  # the parent's own block, untouched by its children
    assert len({pool.get_block_ids(k)[4] for k in kids} | {pool.get_block_ids(root)[4]}) == 6
    pool._allocator.check()


def test_decode_batch_refusals():
    pool = AgentKVPool(config=PoolConfig(total_blocks=16, block_size=4, num_layers=1, num_kv_heads=1, head_dim=16,
                                         dtype="float16", device="cuda"))
    a = pool.create_root([])
    with pytest.raises(ValueError, match="twice"):
        pool.decode_batch([a, a])
    with pytest.raises(ValueError, match="rows"):
        pool.decode_batch([a], rows=0)
    b = pool.decode_batch([a], width=2)
    with pytest.raises(ValueError, match="tokens for 2"):
        b.advance([[1], [2]])
    before = pool.stats()["allocated_blocks"]
    with pytest.raises(ValueError, match="cannot hold"):
        b.advance([[1] * 9])
    assert pool.stats()["allocated_blocks"] == before and a.tokens == []
    b.advance([[1] * 8])
    with pytest.raises(ValueError, match="bounds"):
        b.attend(0, torch.zeros(1, 1, 16, dtype=F16, device=DEV), keep=1)


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_hf_cache_attends_in_place(dtype):
    """store() + attend() against update() and the same attention on what it
    assembles; the prompt in one call, then single tokens, after a fork too."""
    t = {"float16": F16, "float32": F32}[dtype]
    H, G, D, L = 2, 2, 64, 2
    pool = AgentKVPool(config=PoolConfig(total_blocks=64, block_size=8, num_layers=L, num_kv_heads=H, head_dim=D,
                                         dtype=dtype, device="cuda"))
    ours = AgentKVCache(pool, pool.create_root([]))
    theirs = AgentKVCache(pool, pool.create_root([]))
    g = _gen(9)
    for turn, n in enumerate([21, 1, 1, 5, 1]):
        if turn == 2:
            ours, theirs = ours.fork(), theirs.fork()
        for layer in range(L):
            k, v, q = (_randn(g, 1, h, n, D, dtype=t) for h in (H, H, H * G))
            ours.store(k, v, layer)
            ks, vs = theirs.update(k, v, layer)
            out = ours.attend(q, layer)
            total = ks.shape[2]
            x = (q.double().view(1, H, G, n, D) @ ks.double()[:, :, None].transpose(3, 4)) * D ** -0.5
            mask = torch.arange(total, device=DEV) <= torch.arange(total - n, total, device=DEV)[:, None]
            want = torch.softmax(x.masked_fill(~mask, -math.inf), -1) @ vs.double()[:, :, None]
            assert out.shape == (1, H * G, n, D)
            _check(out, want.reshape(1, H * G, n, D), t)
    assert ours.get_seq_length() == theirs.get_seq_length() == 29
    with pytest.raises(ValueError):
        ours.attend(torch.zeros(2, H * G, 1, D, dtype=t, device=DEV), 0)


def _two_agents(**kw):
    pool = AgentKVPool(config=PoolConfig(total_blocks=16, block_size=4, num_layers=1, num_kv_heads=1, head_dim=16,
                                         dtype="float16", device="cuda"))
    agents = [pool.create_root([]) for _ in range(2)]
    return pool, agents, pool.decode_batch(agents, **kw)


def test_append_needs_an_advance():
    """Before one, or behind one that failed, there are no new tokens: the
    agents' last ones must not be written over."""
    x = torch.ones(2, 1, 16, dtype=F16, device=DEV)
    _, _, batch = _two_agents()
    with pytest.raises(RuntimeError, match="advance"):
        batch.append(0, x, x)
    batch.advance([[1], [2]])
    batch.append(0, x, x, check=True)
    with pytest.raises(MemoryError):
        batch.advance([[1], [2] * 100])
    with pytest.raises(RuntimeError, match="advance"):
        batch.append(0, x, x)
    batch.advance([[1], [2]])
    batch.append(0, x, x, check=True)
    assert torch.equal(batch.attend(0, x), x)


def test_a_freed_agent_stops_an_advance_before_anything_changes():
    pool, (a, b), batch = _two_agents()
    batch.advance([[1], [2]])
    pool.free(b)
    with pytest.raises(Exception):
        batch.advance([[1], []])
    assert a.tokens == [1]


def test_a_captured_uneven_step_follows_later_advances():
    """The step's starts are at one address, and those of a later advance of
    one token each are there too."""
    def operands(x):
        return torch.full((6, 1, 16), float(x), dtype=F16, device=DEV)

    pool, agents, batch = _two_agents(width=4)
    batch.advance([[1, 2], [3]])
    k = operands(1)
    batch.append(0, k, k, check=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        batch.append(0, k, k)
    for turn, counts in enumerate(([0, 5], [1, 1], [3, 1])):
        batch.advance([[7] * n for n in counts])
        k.copy_(operands(turn + 2))
        graph.replay()
        torch.cuda.synchronize()
    data = pool._allocator._kv_data
    for agent, want in zip(agents, ([1, 1, 3, 4, 4, 4], [1, 2, 2, 2, 2, 2, 3, 4])):
        ids = pool.get_block_ids(agent)
        got = [data[ids[i // 4], 0, 0, 0, i % 4, 0].item() for i in range(len(agent.tokens))]
        assert got == want


def test_hf_cache_attends_eagerly_after_a_capture():
    """The lengths that a captured call makes exist when it is replayed, not
    before: an eager call makes its own."""
    pool = AgentKVPool(config=PoolConfig(total_blocks=16, block_size=8, num_layers=1, num_kv_heads=1, head_dim=16,
                                         dtype="float16", device="cuda"))
    cache = AgentKVCache(pool, pool.create_root([]))
    g = _gen(4)
    k, v, q = (_randn(g, 1, 1, 5, 16, dtype=F16) for _ in range(3))
    cache.store(k, v, 0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        captured = cache.attend(q, 0)
    eager = cache.attend(q, 0)
    torch.cuda.synchronize()
    x = q.double()[0, 0] @ k.double()[0, 0].T / 4
    x = x.masked_fill(~torch.ones(5, 5, dtype=torch.bool, device=DEV).tril(), -math.inf)
    _check(eager, (torch.softmax(x, 1) @ v.double()[0, 0])[None, None], F16)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured, eager)
