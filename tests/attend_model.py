"""The index arithmetic of k_attend (agentkv_b200/csrc/akv_attend.cu) in
Python: how a batch's chunks are listed, dealt to the CTAs, and which CTA joins
which pieces.  Same names and the same rules, statement by statement where the
result depends on them."""

CHUNK, FAN = 64, 16


def extent(length, width, bs, window, keep):
    n = min(max(length, 0), width * bs)
    lo = n - window if window > 0 and n > window else 0
    if keep:
        taken = min(-(-n // bs), keep) * bs
        return n, lo, 0, -(-taken // CHUNK)
    first = lo // CHUNK
    return n, lo, first, -(-n // CHUNK) - first


def shared_chunks(tables, rows, held, bs):
    """shared_chunks() of the rows given; the four probes of a step at once."""
    live = [s for s in rows if held[s] > 0]
    if len(live) < 2:
        return 0
    hi = min(held[s] // CHUNK for s in live)

    def same(c):
        return len({tables[s][(c * CHUNK - 1) // bs] for s in live}) == 1

    if hi == 0 or not same(1):
        return 0
    lo = 1
    while lo < hi:
        step = (hi - lo + 3) // 4
        probes = [same(min(lo + (i + 1) * step, hi)) for i in range(4)]
        to, stop = lo, hi
        for i in range(4):
            at = min(lo + (i + 1) * step, hi)
            if probes[i] and to == min(lo + i * step, hi):
                to = at
            else:
                stop = min(stop, at - 1)
        assert (to, max(to, stop)) != (lo, hi)  # each step narrows the range
        lo, hi = to, max(to, stop)
    return lo


class Deal:
    def __init__(self, total, grid):
        self.total, self.ctas = total, min(total, grid)

    def begin(self, c):
        return self.total * c // self.ctas

    def cta_of(self, u):
        c = u * self.ctas // self.total
        while self.begin(c + 1) <= u:
            c += 1
        while self.begin(c) > u:
            c -= 1
        return c


def simulate(lengths, tables, width, bs, heads, parts, rows_per, grid, window=0, keep=0):
    """Runs every CTA.  Returns (reads, joins): reads is a list of (row whose
    table is used, rows served, head, part, chunk); joins lists, per pair, the CTAs whose
    pieces were joined.  Asserts that every counter ends at zero."""
    S = len(lengths)
    ext = [extent(n, width, bs, window, keep) for n in lengths]
    groups = [list(range(g, min(g + rows_per, S))) for g in range(0, S, rows_per)]
    held = [e[0] for e in ext]
    front = [0 if window or keep or rows_per == 1 else shared_chunks(tables, g, held, bs) for g in groups]
    chunks = [f + sum(max(0, ext[s][3] - f) for s in g) for f, g in zip(front, groups)]
    pairs = heads * parts
    total = sum(c * pairs for c in chunks)
    reads, joins, arrived, slots = [], {}, {}, {}
    if total == 0:
        return reads, joins
    deal = Deal(total, grid)
    starts = [0]
    for c in chunks:
        starts.append(starts[-1] + c * pairs)
    for cta in range(deal.ctas):
        x, end = deal.begin(cta), deal.begin(cta + 1)
        g = max(i for i in range(len(groups)) if starts[i] <= x and chunks[i])
        rest = x - starts[g]
        while x < end:
            if rest >= chunks[g] * pairs:
                g, rest = g + 1, 0
                continue
            rows, f, size, at = groups[g], front[g], chunks[g], rest
            if f == 0:  # each row by itself
                k = 0
                while at >= ext[rows[k]][3] * pairs:
                    at -= ext[rows[k]][3] * pairs
                    k += 1
                rows, size = rows[k:k + 1], ext[rows[k]][3]
            pair, a = divmod(at, size)
            n = min(end - x, size - a)
            h, part = divmod(pair, parts)
            base, count = 0, len(rows)
            lead = 0
            if f:
                while ext[rows[lead]][0] == 0:
                    lead += 1
            i, differ = (lead - count if f else 0), False
            while i < count:
                r = i + count if i < 0 else i
                n_r, _, first, c_r = ext[rows[r]]
                frm = 0 if i < 0 else f
                length = f if i < 0 else max(0, c_r - f)
                lo, hi = max(a, base), min(a + n, base + length)
                ca, cb = first + frm + lo - base, first + frm + hi - base
                if i < 0 and r == lead and lo < hi:
                    blocks = range(ca * CHUNK // bs, (cb * CHUNK - 1) // bs + 1)
                    live = [s for s in rows if ext[s][0] > 0]
                    differ = any(tables[s][j] != tables[rows[lead]][j] for j in blocks for s in live)
                every = i < 0 and not differ
                if lo < hi and n_r > 0:
                    served = tuple(s for s in rows if ext[s][0] > 0) if every else (rows[r],)
                    reads += [(rows[r], served, h, part, c) for c in range(ca, cb)]
                if i < 0 and (every or i == -1):
                    base, i = f, -1
                elif i >= 0:
                    base += length
                i += 1
            if not (a == 0 and n == size):
                c0, c1 = deal.cta_of(x - a), deal.cta_of(x - a + size - 1)
                assert c0 <= cta <= c1 and c0 < c1
                slot = (cta, cta == c0)
                assert slot not in slots
                name = (rows[0], f > 0, pair, x - a, size)
                slots[slot] = name
                part0 = c0 + (cta - c0) // FAN * FAN
                near = min(FAN, c1 + 1 - part0)
                many = (c1 - c0) // FAN + 1
                assert many <= 2 * FAN
                key = 2 * part0 + (part0 == c0)
                arrived[key] = arrived.get(key, 0) + 1
                if arrived[key] == near:
                    arrived[key] = 0
                    pieces = [part0 + k for k in range(near)]
                    assert all(slots.get((c, c == c0)) == name for c in pieces)
                    if many > 1:
                        key = 2 * grid + c0
                        arrived[key] = arrived.get(key, 0) + 1
                        joins.setdefault(name, []).extend(pieces)
                        if arrived[key] == many:
                            arrived[key] = 0
                    else:
                        joins[name] = pieces
                assert key < 3 * grid
            x, rest = x + n, rest + n
    assert not any(arrived.values())
    for (_, _, _, first, size), ctas in joins.items():
        assert sorted(ctas) == list(range(deal.cta_of(first), deal.cta_of(first + size - 1) + 1))
    assert sum(len(c) for c in joins.values()) == len(slots)
    return reads, joins
