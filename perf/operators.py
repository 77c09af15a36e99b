"""The attention operators over the paged key-value pool: what is measured, and their plain forms.

Three operators on the pool's own layout ``[blocks, layers, 2, kv_heads, block_size, head_dim]``:

* ``append``: a ragged batch's new keys and values go to their pages, the keys rotated by their
  position on the way (the queries of the same tokens too), and each touched page's key bounds
  (the minimum and maximum of its keys by dimension) are brought up to date;
* ``attend``: attention of one new token of each sequence over its pages;
* ``sparse``: the pages that each sequence's key bounds rank highest for the new token, and the
  attention over those pages alone.

``run`` computes them with elementary torch operations, or through ``agentkv_b200.attention``
where ``own`` is true.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}
LARGEST = 1.7976931348623157e308


# ── cases ────────────────────────────────────────────────────────────────────
def _append(name, **kw):
    case = dict(op="append", name=name, dtype="bfloat16", kv_heads=8, group=4, head_dim=128, block=16, layers=2,
                layer=1, rows=1, empty=0, old_lo=0, old_hi=0, new_lo=1, new_hi=1, rotary=128, interleaved=False)
    case.update(kw)
    return case


def _attend(name, **kw):
    case = dict(op="attend", name=name, dtype="bfloat16", kv_heads=8, group=4, head_dim=128, block=16, layers=2,
                layer=1, rows=1, empty=0, lo=1, hi=1, shared=0, window=0)
    case.update(kw)
    return case


def _sparse(name, **kw):
    case = dict(op="sparse", name=name, dtype="bfloat16", kv_heads=8, group=4, head_dim=128, block=16, layers=1,
                layer=0, rows=1, empty=0, lo=1, hi=1, keep=64, first=1, last=2)
    case.update(kw)
    return case


def listed():
    return [
        # one agent's decode step: one token of one sequence, where only latency counts
        _append("append one token", old_lo=1000, old_hi=1000),
        # a serving batch's decode step, padded at its end as a captured step is; pairs of neighbours rotated
        _append("append 256 rows", dtype="float16", rows=256, empty=9, old_lo=0, old_hi=8000, interleaved=True),
        # prompts of several agents arriving together, uneven, some of them behind a cached prefix
        _append("append prompts", rows=6, old_lo=0, old_hi=2000, new_lo=411, new_hi=2411),
        # a small model in 32 bits with a partly rotated head of an odd size, in chunks of some tokens
        _append("append chunks fp32", dtype="float32", kv_heads=2, group=3, head_dim=80, rotary=32, rows=37, old_lo=0,
                old_hi=900, new_lo=1, new_hi=33),
        # one agent, a short context: latency
        _attend("attend one short", dtype="float16", lo=517, hi=517),
        # one agent over a very long context: the split over the length
        _attend("attend one long", group=8, lo=200001, hi=200001, layers=1, layer=0),
        # a serving batch of uneven lengths, padded at its end
        _attend("attend 32 uneven", rows=32, empty=2, lo=1, hi=16383),
        # a large serving batch: bandwidth
        _attend("attend 256", rows=256, lo=3900, hi=4292, layers=1, layer=0),
        # the children of a Tree-of-Thought fan-out: one shared prompt of 256 pages, some own pages each
        _attend("attend 64 children", rows=64, lo=4100, hi=4240, shared=256),
        # a small model in 32 bits with a sliding window, over smaller pages
        _attend("attend window fp32", dtype="float32", kv_heads=4, group=2, head_dim=64, block=8, rows=48, empty=1, lo=1,
                hi=5000, window=1024),
        # one agent over a long context through its best 128 of 8,126 pages
        _sparse("sparse one long", lo=130001, hi=130001, keep=128),
        # a serving batch of long contexts
        _sparse("sparse 32 rows", rows=32, lo=9000, hi=32768, keep=160, first=1, last=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "sparse"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    case = dict(dtype=dtype, kv_heads=rng.choice([1, 2, 4, 5, 8]), group=rng.choice([1, 2, 3, 4, 6, 8, 16]),
                head_dim=rng.choice([64, 64, 80, 96, 128, 128, 128, 256]), block=rng.choice([8, 16, 16, 16, 32, 64]),
                layers=2, layer=rng.randrange(2))
    width = case["kv_heads"] * case["head_dim"]
    if op == "append":
        case["rows"] = _log(rng, 1, 300)
        case["empty"] = rng.choice([0, 0, min(3, case["rows"] - 1)])
        tokens = max(1, min(2000, 4_000_000 // (width * (2 + case["group"])) // case["rows"]))
        case.update(old_lo=0, old_hi=_log(rng, 1, 9000), new_lo=1, new_hi=rng.choice([1, 1, _log(rng, 1, tokens)]),
                    rotary=rng.choice([case["head_dim"], case["head_dim"], case["head_dim"] // 2]),
                    interleaved=rng.random() < 0.5)
        return dict(op="append", **case)
    case["rows"] = _log(rng, 1, 256)
    case["empty"] = rng.choice([0, 0, min(2, case["rows"] - 1)])
    most = max(64, min(160_000, 400_000_000 // width // case["rows"]))
    hi = _log(rng, 17, most)
    case.update(lo=rng.choice([1, max(1, hi // 2), hi]), hi=hi)
    if op == "attend":
        shared = rng.choice([0, 0, 0, case["lo"] // case["block"]])
        case.update(shared=shared, window=rng.choice([0, 0, 0, _log(rng, 1, hi)]))
        return dict(op="attend", **case)
    case["layers"], case["layer"] = 1, 0
    first, last = rng.choice([0, 1, 2]), rng.choice([1, 2, 4])
    case.update(keep=max(first + last, _log(rng, 4, 400)), first=first, last=last)
    return dict(op="sparse", **case)


# ── inputs ───────────────────────────────────────────────────────────────────
def _spread(lo, hi, rows, empty):
    """`rows` whole numbers from lo to hi in a scrambled order, the last `empty` of them 0."""
    n = rows - empty
    step = next(s for s in (7919, 7907, 7901, 7883) if math.gcd(s, n) == 1)
    return [lo + (i * step % n) * (hi - lo) // max(n - 1, 1) for i in range(n)] + [0] * empty


def _lengths(case):
    """(tokens held before the call, new tokens) of each row."""
    if case["op"] == "append":
        old = _spread(case["old_lo"], case["old_hi"], case["rows"], case["empty"])
        new = _spread(case["new_lo"], case["new_hi"], case["rows"], case["empty"])
        return old, new
    return _spread(case["lo"], case["hi"], case["rows"], case["empty"]), [0] * case["rows"]


def _randn(gen, *shape, dtype):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype)


def _pages(pages, gen, total):
    """Page ids in a shuffled order, as a pool that has been in use hands them out."""
    return torch.randperm(total, generator=gen, device=DEVICE)[:pages].to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed * 1009 + 17)
    dtype, H, G, D, bs = DTYPES[case["dtype"]], case["kv_heads"], case["group"], case["head_dim"], case["block"]
    old, new = _lengths(case)
    lens = [o + n for o, n in zip(old, new)]
    S = len(lens)
    st = dict(case=case, lengths=torch.tensor(lens, dtype=torch.int32, device=DEVICE))
    need = [-(-n // bs) for n in lens]
    W = max(max(need), 1)
    st["width"] = W
    if case["op"] == "append":
        # the pages that the new tokens touch are each row's own; the full ones before them are drawn from a
        # small set, since nothing reads them here
        first = [o // bs for o in old]
        own_pages = [max(0, e - f) if n else 0 for e, f, n in zip(need, first, new)]
        total = sum(own_pages) + 32
        ids = _pages(total, gen, total).cpu()
        table, at = torch.zeros((S, W), dtype=torch.int32), 32
        for s in range(S):
            table[s, :first[s]] = ids[:32][torch.arange(first[s]) % 32]
            if own_pages[s]:
                table[s, first[s]:need[s]] = ids[at:at + own_pages[s]]
                at += own_pages[s]
        T = sum(new)
        st["tables"] = table.to(DEVICE)
        st["pool"] = _randn(gen, total, case["layers"], 2, H, bs, D, dtype=dtype)
        st["bounds"] = torch.zeros((total, case["layers"], H, 2, D), dtype=dtype, device=DEVICE)
        st["key"], st["value"] = _randn(gen, T, H, D, dtype=dtype), _randn(gen, T, H, D, dtype=dtype)
        st["query"] = _randn(gen, T, H * G, D, dtype=dtype)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        st["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEVICE)
        angles = _angles(torch.arange(max(lens), dtype=torch.float64, device=DEVICE), case["rotary"])
        st["rope"] = torch.cat([angles.cos(), angles.sin()], 1).to(torch.float32)
        # what a program that computes the plain form lays out of its batch beforehand
        rows = torch.tensor(new, device=DEVICE)
        st["row"] = torch.repeat_interleave(torch.arange(S, device=DEVICE), rows, output_size=T)
        st["touched"] = torch.tensor([(s, p) for s in range(S) if new[s] for p in range(first[s], need[s])],
                                     dtype=torch.int64, device=DEVICE).reshape(-1, 2)
        return st
    shared = case.get("shared", 0)
    own_pages = [max(0, n - shared) for n in need]
    total = shared + sum(own_pages) + 3
    ids = _pages(total, gen, total).cpu()
    table, at = torch.zeros((S, W), dtype=torch.int32), shared
    for s in range(S):
        if need[s]:
            table[s, :min(shared, need[s])] = ids[:min(shared, need[s])]
            table[s, shared:need[s]] = ids[at:at + own_pages[s]]
            at += own_pages[s]
    st["tables"] = table.to(DEVICE)
    pool = _randn(gen, total, case["layers"], 2, H, bs, D, dtype=dtype)
    if case["op"] == "sparse":
        # the keys of a page resemble one another, as neighbouring tokens' do: a centre of the page's own
        centre = _randn(gen, total, case["layers"], 1, H, 1, D, dtype=dtype)
        pool[:, :, :1].mul_(0.6).add_(centre, alpha=0.8)
        st["bounds"] = torch.stack([pool[:, :, 0].amin(3), pool[:, :, 0].amax(3)], 3)
        tail = [(s, need[s] - 1, lens[s] - (need[s] - 1) * bs) for s in range(S) if lens[s] % bs]
        if tail:  # of a page that is not full, the keys that it has
            s, p, n = (torch.tensor(x, device=DEVICE) for x in zip(*tail))
            page = st["tables"][s, p].long()
            k = pool[page, :, 0]
            k = torch.where((torch.arange(bs, device=DEVICE) < n[:, None])[:, None, None, :, None], k, k[..., :1, :])
            st["bounds"][page] = torch.stack([k.amin(3), k.amax(3)], 3)
        st["bounds"] = st["bounds"].contiguous()
    st["pool"] = pool
    st["query"] = _randn(gen, S, H * G, D, dtype=dtype).mul_(1.5)
    st["scale"] = 1.0 / math.sqrt(D)
    return st


def _angles(positions, rotary):
    """Angles [positions, rotary / 2] in 64 bits."""
    inverse = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=positions.device) / rotary)
    return positions[:, None] * inverse


# ── the plain forms ──────────────────────────────────────────────────────────
def _rotated(x, cos, sin, rotary, interleaved):
    """x [T, heads, D] with its first `rotary` dimensions rotated by pairs."""
    a = x[..., :rotary]
    cos, sin = cos[:, None], sin[:, None]
    if interleaved:
        u, v = a[..., 0::2], a[..., 1::2]
        r = torch.stack([u * cos - v * sin, v * cos + u * sin], -1).flatten(-2)
    else:
        u, v = a[..., :rotary // 2], a[..., rotary // 2:]
        r = torch.cat([u * cos - v * sin, v * cos + u * sin], -1)
    return torch.cat([r, x[..., rotary:]], -1)


def _plain_append(st):
    c, pool, bounds = st["case"], st["pool"], st["bounds"]
    bs, rot, layer, dtype = c["block"], c["rotary"], c["layer"], st["pool"].dtype
    lengths, starts, row, tables = st["lengths"].long(), st["starts"].long(), st["row"], st["tables"].long()
    at = torch.arange(row.numel(), device=row.device)
    pos = lengths[row] - starts[row + 1] + at
    cs = st["rope"][pos]
    cos, sin = cs[:, :rot // 2], cs[:, rot // 2:]
    page = tables[row, pos // bs]
    pool[page, layer, 0, :, pos % bs] = _rotated(st["key"].float(), cos, sin, rot, c["interleaved"]).to(dtype)
    pool[page, layer, 1, :, pos % bs] = st["value"]
    query = _rotated(st["query"].float(), cos, sin, rot, c["interleaved"]).to(dtype)
    s, p = st["touched"].unbind(1)
    page = tables[s, p]
    keys = pool[page, layer, 0].float()
    held = (torch.arange(bs, device=row.device) < (lengths[s] - p * bs)[:, None])[:, None, :, None]
    bounds[page, layer, :, 0] = torch.where(held, keys, math.inf).amin(2).to(dtype)
    bounds[page, layer, :, 1] = torch.where(held, keys, -math.inf).amax(2).to(dtype)
    return {"pool": pool, "bounds": bounds, "query": query}


def _plain_attend(query, keys, values, held, scale):
    """query [S, H, G, D], keys and values [S, H, n, D] in 32 bits, held [S, 1 or H, 1, n]."""
    scores = torch.where(held, (query @ keys.transpose(2, 3)) * scale, -math.inf)
    top = scores.amax(3, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = weights.sum(3, keepdim=True)
    out = weights @ values
    return torch.where(total > 0, out / total, 0.0)


def _plain_dense(st):
    c, pool = st["case"], st["pool"]
    S, H, G, D, bs, W = c["rows"], c["kv_heads"], c["group"], c["head_dim"], c["block"], st["width"]
    data = pool[st["tables"].long(), c["layer"]]
    keys = data[:, :, 0].permute(0, 2, 1, 3, 4).reshape(S, H, W * bs, D).float()
    values = data[:, :, 1].permute(0, 2, 1, 3, 4).reshape(S, H, W * bs, D).float()
    pos, length = torch.arange(W * bs, device=pool.device), st["lengths"][:, None]
    held = pos < length
    if c["window"]:
        held = held & (pos >= length - c["window"])
    out = _plain_attend(st["query"].view(S, H, G, D).float(), keys, values, held[:, None, None], st["scale"])
    return {"out": out.to(pool.dtype).view(S, H * G, D)}


def _ranked(score, pages, keep, first, last):
    """The selected page positions [S, H, keep] of scores [S, H, W]: all of a row that has no more than `keep`; else
    its first and last pages and the highest of the rest, the lowest position of equal ones. Ascending, -1 behind."""
    S, H, W = score.shape
    at = torch.arange(W, device=score.device)
    n = pages[:, None, None]
    score = torch.where(score.isnan(), LARGEST, score).clamp(-LARGEST, LARGEST)
    score = torch.where((at < first) | (at >= n - last), math.inf, score)
    score = torch.where(at < n, score, -math.inf)
    order = torch.sort(score, dim=2, descending=True, stable=True).indices[..., :keep]
    order = torch.where(order < n, order, W).sort(2).values
    order = torch.where(order < W, order, -1).to(torch.int32)
    return torch.nn.functional.pad(order, (0, keep - order.shape[2]), value=-1)


def _plain_sparse(st):
    c, pool = st["case"], st["pool"]
    S, H, G, D, bs = c["rows"], c["kv_heads"], c["group"], c["head_dim"], c["block"]
    tables, lengths, layer = st["tables"].long(), st["lengths"].long(), c["layer"]
    # 64 bits: which of two pages is taken hangs on their scores' last places
    query = st["query"].view(S, H, G, D).double()
    up, down = query.clamp(min=0).sum(2), query.clamp(max=0).sum(2)
    box = st["bounds"][tables, layer].double()
    score = (box[:, :, :, 1] * up[:, None] + box[:, :, :, 0] * down[:, None]).sum(3).transpose(1, 2)
    selected = _ranked(score, (lengths + bs - 1) // bs, c["keep"], c["first"], c["last"])
    taken = selected.long()
    page = torch.gather(tables[:, None].expand(S, H, -1), 2, taken.clamp(min=0))
    head = torch.arange(H, device=pool.device)[:, None]
    n = c["keep"] * bs
    keys = pool[page, layer, 0, head].reshape(S, H, n, D).float()
    values = pool[page, layer, 1, head].reshape(S, H, n, D).float()
    pos = taken[..., None] * bs + torch.arange(bs, device=pool.device)
    held = ((taken >= 0)[..., None] & (pos < lengths[:, None, None, None])).reshape(S, H, 1, n)
    out = _plain_attend(query.float(), keys, values, held, st["scale"])
    return {"selected": selected, "out": out.to(pool.dtype).view(S, H * G, D)}


# ── one pass ─────────────────────────────────────────────────────────────────
def run(st):
    c = st["case"]
    if not own:
        return {"append": _plain_append, "attend": _plain_dense, "sparse": _plain_sparse}[c["op"]](st)
    from agentkv_b200 import attention as A

    pool, layer, tables, lengths = st["pool"], c["layer"], st["tables"], st["lengths"]
    if c["op"] == "append":
        query = A.kv_append(pool, layer, st["key"], st["value"], tables, lengths, starts=st["starts"], rope=st["rope"],
                            interleaved=c["interleaved"], query=st["query"], bounds=st["bounds"])
        return {"pool": pool, "bounds": st["bounds"], "query": query}
    if c["op"] == "attend":
        return {"out": A.paged_attention(st["query"], pool, layer, tables, lengths, scale=st["scale"],
                                         window=c["window"])}
    selected = A.select_blocks(st["query"], st["bounds"], layer, tables, lengths, c["keep"], block_size=c["block"],
                               first=c["first"], last=c["last"])
    return {"selected": selected, "out": A.paged_attention(st["query"], pool, layer, tables, lengths,
                                                           scale=st["scale"], selected=selected)}


def work(case):
    e, H, G, D, bs = BYTES[case["dtype"]], case["kv_heads"], case["group"], case["head_dim"], case["block"]
    old, new = _lengths(case)
    S = case["rows"]
    if case["op"] == "append":
        T = sum(new)
        touched = sum(-(-(o + n) // bs) - o // bs for o, n in zip(old, new) if n)
        # the keys that a first page holds already are read for its bounds
        before = sum(o % bs for o, n in zip(old, new) if n)
        read = T * (2 + G) * H * D * e + before * H * D * e + T * case["rotary"] * 4 + touched * 4
        return {"bytes": read + T * (2 + G) * H * D * e + touched * 2 * H * D * e,
                "flops": T * (1 + G) * H * case["rotary"] * 3 + (T + before) * 2 * H * D}
    io = 2 * S * H * G * D * e
    pages = [-(-n // bs) for n in old]
    if case["op"] == "attend":
        shared = case["shared"] * bs
        seen = [min(n, case["window"] or n) for n in old]
        common = max([min(n, shared) - (n - v) for n, v in zip(old, seen)] + [0])
        rest = sum(v - max(0, min(n, shared) - (n - v)) for n, v in zip(old, seen))
        return {"bytes": (common + rest) * H * 2 * D * e + io + sum(pages) * 4, "flops": sum(seen) * H * G * D * 4}
    taken = [min(p, case["keep"]) for p in pages]
    full = [min(n, t * bs) for n, t in zip(old, taken)]
    scored = sum(p for p in pages if p > case["keep"])
    return {"bytes": scored * H * 2 * D * e + sum(full) * H * 2 * D * e + io + sum(pages) * 4 + S * H * case["keep"] * 4,
            "flops": scored * H * 4 * D + sum(full) * H * G * D * 4}


# ── the definition in 64 bits ────────────────────────────────────────────────
def exact(case, seed):
    st = prepare(case, seed)
    H, G, D, bs, layer = case["kv_heads"], case["group"], case["head_dim"], case["block"], case["layer"]
    old, new = _lengths(case)
    table = st["tables"].cpu().tolist()
    pool = st["pool"]
    if case["op"] == "append":
        rot = case["rotary"]
        if case["interleaved"]:
            left, right = range(0, rot, 2), range(1, rot, 2)
        else:
            left, right = range(rot // 2), range(rot // 2, rot)
        left, right = torch.tensor(left, device=DEVICE), torch.tensor(right, device=DEVICE)
        pool, bounds = pool.double(), st["bounds"].double()
        query, key, value = st["query"].double(), st["key"].double(), st["value"].double()
        at = 0
        for s, (o, n) in enumerate(zip(old, new)):
            if not n:
                continue
            turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEVICE),
                               _angles(torch.arange(o, o + n, dtype=torch.float64, device=DEVICE), rot))[:, None]
            for x in (query, key):
                y = torch.complex(x[at:at + n][..., left], x[at:at + n][..., right]) * turn
                x[at:at + n, :, left], x[at:at + n, :, right] = y.real, y.imag
            for p in range(o // bs, -(-(o + n) // bs)):
                lo, hi = max(o, p * bs), min(o + n, (p + 1) * bs)
                b = table[s][p]
                pool[b, layer, 0, :, lo - p * bs:hi - p * bs] = key[at + lo - o:at + hi - o].transpose(0, 1)
                pool[b, layer, 1, :, lo - p * bs:hi - p * bs] = value[at + lo - o:at + hi - o].transpose(0, 1)
                held = pool[b, layer, 0, :, :hi - p * bs]
                bounds[b, layer, :, 0], bounds[b, layer, :, 1] = held.min(1).values, held.max(1).values
            at += n
        return {"pool": pool, "bounds": bounds, "query": query}
    S = case["rows"]
    out = torch.zeros((S, H * G, D), dtype=torch.float64, device=DEVICE)
    selected = torch.full((S, H, case.get("keep", 1)), -1, dtype=torch.int32)
    for s, n in enumerate(old):
        if not n:
            continue
        pages = -(-n // bs)
        ids = st["tables"][s, :pages].long()
        q = st["query"][s].double().view(H, G, 1, D)
        if case["op"] == "attend":
            lo = max(0, n - case["window"]) if case["window"] else 0
            p0 = lo // bs
            kv = pool[ids[p0:], layer].double().permute(1, 2, 0, 3, 4).reshape(2, H, 1, -1, D)[:, :, :,
                                                                                              lo - p0 * bs:n - p0 * bs]
            w = torch.softmax((q * st["scale"] @ kv[0].transpose(2, 3)), 3)
            out[s] = (w @ kv[1]).reshape(H * G, D)
            continue
        keep = min(case["keep"], pages)
        box = st["bounds"][ids, layer].double()
        best = torch.maximum(q * box[:, :, 0].transpose(0, 1)[:, None], q * box[:, :, 1].transpose(0, 1)[:, None])
        score = best.sum((1, 3)).cpu().tolist()
        for h in range(H):
            always = [p for p in range(pages) if p < case["first"] or p >= pages - case["last"]]
            if keep == pages:
                taken = list(range(pages))
            else:
                rest = sorted(set(range(pages)) - set(always), key=lambda p: (-score[h][p], p))
                taken = sorted(always + rest[:keep - len(always)])
            selected[s, h, :keep] = torch.tensor(taken, dtype=torch.int32)
            at = torch.tensor(taken, device=DEVICE)
            kv = pool[ids[at], layer][:, :, h].double()
            k, v = kv[:, 0].reshape(-1, D), kv[:, 1].reshape(-1, D)
            held = (at[:, None] * bs + torch.arange(bs, device=DEVICE)).reshape(-1) < n
            w = torch.softmax(q[h, :, 0] * st["scale"] @ k[held].T, 1)
            out[s, h * G:(h + 1) * G] = w @ v[held]
    if case["op"] == "attend":
        return {"out": out}
    return {"selected": selected.to(DEVICE), "out": out}
