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
