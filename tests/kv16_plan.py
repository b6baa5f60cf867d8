"""The prompts' kernel deals the items of a launch out in waves where its keys do not fit in the L2 cache; restated, item by item, so
that tests know which parts of that plan their batches reach."""

KV_TILE, ITEM_TILES, L2_BYTES, PLAN_REQS = 128, 2, 48 << 20, 4096


class Plan:
    """`waves` of whole items; `shares[c]`: what CTA c gets of the rest, in KV tiles; `skipped`: items of the rest whose pieces lie on
    both sides of a CTA without a share."""

    def __init__(self, kv_lens, q_lens, Hq, Hkv, D, sms):
        G, rows, C = Hq // Hkv, 256 if D == 128 else 128, sms * (2 if D == 64 else 1)
        lengths, tiles = [], 0
        for n, q in zip(kv_lens, q_lens):
            if n == 0 or q == 0:
                continue
            t = -(-n // KV_TILE)
            tiles += t
            lengths += [t + ITEM_TILES] * (-(-q * G // rows) * Hkv)
        self.items = len(lengths)
        in_waves = tiles * Hkv * KV_TILE * D * 4 > L2_BYTES and len(lengths) >= 2 * C and len(kv_lens) <= PLAN_REQS
        self.waves = len(lengths) // C - 1 if in_waves else 0
        self.shares, self.skipped = [], 0
        if not in_waves:
            return
        first = self.waves * C
        loads = [sum(lengths[c:first:C]) for c in range(C)]
        work = sum(lengths[first:])
        level = sum(lengths) // C
        while sum(max(0, level - x) for x in loads) < work:
            level += 1
        at = 0
        for x in loads:
            share = min(max(0, level - x), work - at)
            self.shares.append(share)
            at += share
        ends = [sum(self.shares[:c + 1]) for c in range(C)]

        def owner(x):
            return next(c for c in range(C) if x < ends[c])
        at = 0
        for n in lengths[first:]:
            a, b = owner(at + ITEM_TILES), owner(at + n - 1)
            self.skipped += any(self.shares[c] == 0 for c in range(a + 1, b))
            at += n
