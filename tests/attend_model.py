"""The index arithmetic of k_attend (agentkv_b200/csrc/akv_attend.cu) in
Python: how a batch's chunks are dealt to the CTAs, and which CTA joins which
pieces.  Same names and the same rules, statement by statement where the result
depends on them."""

CHUNK, FAN, LEAST = 64, 20, 2


def extent(length, width, bs, window, keep):
    n = min(max(length, 0), width * bs)
    lo = n - window if window > 0 and n > window else 0
    if keep:
        taken = min(-(-n // bs), keep) * bs
        return n, lo, 0, -(-taken // CHUNK)
    first = lo // CHUNK
    return n, lo, first, -(-n // CHUNK) - first


def taking_part(n, lo, pos, count):
    """The bits of the `count` positions from pos that lie in [lo, n)."""
    low = max(0, min(count, lo - pos))
    high = max(low, min(count, n - pos))
    return ((1 << high) - 1) & ~((1 << low) - 1)


class Deal:
    def __init__(self, total, grid):
        self.total, self.ctas = total, min(grid, -(-total // LEAST))

    def begin(self, c):
        return self.total * c // self.ctas

    def cta_of(self, u):
        c = u * self.ctas // self.total
        while self.begin(c + 1) <= u:
            c += 1
        while self.begin(c) > u:
            c -= 1
        return c


def simulate(lengths, width, bs, heads, parts, grid, window=0, keep=0):
    """Runs every CTA.  Returns (reads, joins): reads lists (row, head, part,
    chunk); joins, per pair that crosses CTAs, the CTAs whose pieces were joined.  Asserts that
    every piece is written once, joined by the one CTA that comes last, and
    that every counter ends at zero."""
    ext = [extent(n, width, bs, window, keep) for n in lengths]
    pairs = heads * parts
    units = [e[3] * pairs for e in ext]
    total = sum(units)
    reads, joins, arrived, slots = [], {}, {}, {}
    if total == 0:
        return reads, joins
    deal = Deal(total, grid)
    starts = [0]
    for u in units:
        starts.append(starts[-1] + u)
    for cta in range(deal.ctas):
        x, end = deal.begin(cta), deal.begin(cta + 1)
        s = max(i for i in range(len(lengths)) if starts[i] <= x and units[i])
        rest = x - starts[s]
        while x < end:
            chunks = ext[s][3]
            if rest >= units[s]:
                s, rest = s + 1, 0
                continue
            pair, a = divmod(rest, chunks)
            n = min(end - x, chunks - a)
            reads += [(s, *divmod(pair, parts), ext[s][2] + a + i) for i in range(n)]
            if not (a == 0 and n == chunks):
                c0, c1 = deal.cta_of(x - a), deal.cta_of(x - a + chunks - 1)
                assert c0 <= cta <= c1 and c0 < c1 < grid
                slot = 2 * cta + (cta == c0)
                assert slot not in slots and slot < 2 * grid
                slots[slot] = (s, pair)
                first = c0 + (cta - c0) // FAN * FAN
                near = min(FAN, c1 + 1 - first)
                many = (c1 - c0) // FAN + 1
                assert many <= 2 * FAN  # what the joining CTA has room for
                key = 2 * first + (first == c0)
                assert key < 2 * grid
                arrived[key] = arrived.get(key, 0) + 1
                if arrived[key] == near:
                    arrived[key] = 0
                    pieces = [first + k for k in range(near)]
                    assert all(slots.get(2 * c + (c == c0)) == (s, pair) for c in pieces)
                    if many == 1:
                        joins[(s, pair)] = pieces
                    else:
                        key = 2 * grid + c0
                        assert key < 3 * grid
                        arrived[key] = arrived.get(key, 0) + 1
                        joins.setdefault((s, pair), []).extend(pieces)
                        if arrived[key] == many:
                            arrived[key] = 0
            x, rest = x + n, rest + n
    assert not any(arrived.values())
    for (s, pair), ctas in joins.items():
        u = starts[s] + pair * ext[s][3]
        assert sorted(ctas) == list(range(deal.cta_of(u), deal.cta_of(u + ext[s][3] - 1) + 1))
    assert sum(len(c) for c in joins.values()) == len(slots)
    return reads, joins
