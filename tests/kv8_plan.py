"""The schedule of the 8-bit cache's kernel for prompts, as the kernel computes it (``kv8_tall_kernel.cu``: row_tile8, units8, TallWalk8)."""
TILE, ITEM_TILES = 128, 3


class Request:
    def __init__(self, seq, q_len, most_q, group, rows, window, causal, most_keys):
        self.tokens, self.pos0 = min(q_len, most_q), seq - q_len
        self.low = lambda pos: max(0, max(pos, -1) - window + 1) if window else 0
        self.high = lambda pos: max(0, min(pos + 1 if causal else seq, most_keys))
        self.group, self.rows, self.causal = group, rows, causal
        self.lo, self.hi = self.low(self.pos0), self.high(self.pos0 + self.tokens - 1)
        n = self.tokens * group
        self.row_tiles = -(-n // rows)
        self.tiles = -(-self.hi // TILE) - self.lo // TILE if self.hi > self.lo and n > 0 else 0
        self.pairs = self.pair = self.middle = self.head = 0
        if self.tiles:
            n = self.row_tiles
            self.pairs = n // 2
            if n >= 2:
                self.pair = self.tile(0)[2] + self.tile(n - 1)[2]
            if n >= 4:
                self.pair = max(self.pair, self.tile(1)[2] + self.tile(n - 2)[2])
            self.pair += 2 * ITEM_TILES
            if n % 2:
                self.middle = self.tile(n // 2)[2] + ITEM_TILES
            self.head = self.pairs * self.pair + self.middle

    def tile(self, rt):
        rows = self.tokens * self.group
        lo = self.low(self.pos0 + rt * self.rows // self.group)
        hi = self.high(self.pos0 + (min(rows, (rt + 1) * self.rows) - 1) // self.group) if self.causal else self.hi
        return lo, hi, max(1, -(-hi // TILE) - lo // TILE)


def plan(seqs, q_lens, *, ctas, heads, group, rows, window=0, causal=True, most_q=None, most_keys=1 << 30):
    """Pieces of every CTA: (request, head, row tile, first tile, tiles, begins, ends, first CTA, last CTA)."""
    reqs = [Request(s, q, most_q or max(q_lens), group, rows, window, causal, most_keys) for s, q in zip(seqs, q_lens)]
    work = sum(r.head * heads for r in reqs)
    runs = min(ctas, max(work, 1))
    owner = lambda x: ((x + 1) * runs - 1) // work
    out = []
    for cta in range(ctas):
        pieces = []
        at, end = (work * cta // runs, work * (cta + 1) // runs) if cta < runs else (work, work)
        start = r = 0
        while at < end:
            while at >= start + reqs[r].head * heads:
                start += reqs[r].head * heads
                r += 1
            s = reqs[r]
            head = (at - start) // s.head
            base = start + head * s.head
            middle = at - base >= s.pairs * s.pair
            pair = s.pairs if middle else (at - base) // s.pair
            base += pair * s.pair
            length, a = (s.middle if middle else s.pair), at - base
            rt, first, to = pair, 0, length
            t = s.tile(rt)
            if not middle:
                split = min(length - 1, t[2] + ITEM_TILES)
                if a >= split:
                    rt = s.row_tiles - 1 - pair
                    t, first = s.tile(rt), split
                else:
                    to = split
            b = min(to, a + end - at)
            at += b - a
            tile, stop = max(0, a - first - ITEM_TILES), t[2] if b == to else min(t[2], b - first - ITEM_TILES)
            if stop <= tile:
                continue
            pieces.append((r, head, rt, tile, stop - tile, tile == 0, stop == t[2], owner(base + min(first + ITEM_TILES, to - 1)),
                           owner(base + min(first + ITEM_TILES + t[2], to) - 1)))
        out.append(pieces)
    return reqs, out
