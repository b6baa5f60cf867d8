"""The steps of a prompt's pieces that some of their rows do not see whole, as ``kv8_tall_kernel.cu`` counts them (edges8): all others are
seen by every row, and these are few enough for the places that the kernel keeps for notes on their keys."""
import random

import pytest

from tests.kv8_plan import TILE, plan

STEP, PLACES = 64, {128: 8, 256: 12}


@pytest.mark.parametrize("seed", range(200))
def test_steps_that_are_not_whole(seed):
    rng = random.Random(seed)
    group, rows, causal = rng.choice((1, 4, 6, 64)), rng.choice((128, 256)), rng.random() < 0.8
    q = [rng.choice((1, rng.randint(1, 40), rng.randint(1, 3000))) for _ in range(rng.randint(1, 8))]
    kv = [max(0, x + rng.choice((0, rng.randint(0, 200), rng.randint(0, 20000), -rng.randint(0, 50)))) for x in q]
    reqs, ctas = plan(kv, q, ctas=rng.choice((1, 7, 148, 296)), heads=2, group=group, rows=rows, window=rng.choice((0, 0, 1, 63, 100, 1000)), causal=causal)
    for r, _, rt, tile, tiles, *_ in (piece for pieces in ctas for piece in pieces):
        s = reqs[r]
        lo, hi, _ = s.tile(rt)
        key0 = (lo // TILE + tile) * TILE
        steps = max(1, -(-min(tiles * TILE, hi - key0) // STEP))
        first, last = s.pos0 + rt * rows // group, s.pos0 + (min(s.tokens * group, (rt + 1) * rows) - 1) // group
        whole_lo, whole_hi = s.low(last), max(0, first + 1) if causal else 1 << 31
        below = min(steps, -(-max(0, whole_lo - key0) // STEP))
        begin = min(steps, max(below, max(0, whole_hi - key0) // STEP))
        assert below + steps - begin <= PLACES[rows]
        for step in range(below, begin):
            key = key0 + step * STEP
            for pos in range(first, last + 1):
                assert key >= s.low(pos) and (not causal or key + STEP <= pos + 1)


@pytest.mark.parametrize("seed", range(50))
def test_tiles_of_few_rows_that_are_not_whole(seed):
    """The kernel of few rows (``kv8_short_kernel.cu``: Masks): tiles that some of a piece's rows see and some do not see whole, four at most."""
    rng = random.Random(seed)
    for _ in range(200):
        tokens, top = rng.randint(1, 32), rng.choice((-20, 0, 5, rng.randint(0, 3000)))
        window, causal = rng.choice((0, 1, 31, 100, 128, 1000)), rng.random() < 0.8
        low = lambda pos: max(0, max(pos, -1) - window + 1) if window else 0
        bottom = top + tokens - 1
        lo, first = low(bottom), low(top)
        hi, last = (top + 1, bottom + 1) if causal else (1 << 31, 1 << 31)
        key0 = rng.randrange(0, 2000, 32)   # of the piece: a grain of 32 keys
        tiles = [k for k in range(key0, 5000, TILE) if (k < lo or k + TILE > hi) and k < last and k + TILE > first]
        assert len(tiles) <= 4
