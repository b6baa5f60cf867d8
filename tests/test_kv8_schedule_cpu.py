"""The schedule of the 8-bit cache's kernel for prompts: every KV tile of every row tile once, in pieces whose CTAs know one another."""
import random

import pytest

from tests.kv8_plan import ITEM_TILES, plan


def _check(seqs, q_lens, **kw):
    reqs, ctas = plan(seqs, q_lens, **kw)
    seen = {}
    for cta, pieces in enumerate(ctas):
        slots = []
        for r, head, rt, tile, tiles, begins, ends, first, last in pieces:
            seen.setdefault((r, head, rt), []).append((cta, tile, tiles, first, last))
            if not (begins and ends):
                slots.append(begins)
        assert len(slots) == len(set(slots)), "a CTA has one place for a piece that begins a row tile and one for another"
    for r, s in enumerate(reqs):
        for head in range(kw["heads"]):
            for rt in range(s.row_tiles if s.tiles else 0):
                parts = sorted(seen.pop((r, head, rt)))
                at = 0
                for cta, tile, tiles, first, last in parts:
                    assert tile == at and tiles > 0
                    at += tiles
                assert at == s.tile(rt)[2]
                # the CTAs between the first and the last are those that have pieces
                assert [p[0] for p in parts] == list(range(parts[0][3], parts[0][4] + 1)) and len({p[3:] for p in parts}) == 1
    assert not seen
    return ctas


@pytest.mark.parametrize("seed", range(150))
def test_random_launches(seed):
    rng = random.Random(seed)
    n = rng.randint(1, 12)
    q = [rng.choice((0, 1, rng.randint(1, 40), rng.randint(1, 3000))) for _ in range(n)]
    kv = [max(0, x + rng.choice((0, 0, rng.randint(0, 200), rng.randint(0, 20000), -rng.randint(0, 50)))) for x in q]
    _check(kv, q, ctas=rng.choice((1, 7, 148, 296)), heads=rng.choice((1, 2, 8)), group=rng.choice((1, 4, 6, 64)), rows=rng.choice((128, 256)),
           window=rng.choice((0, 0, 1, 100, 1000)), causal=rng.random() < 0.8, most_q=rng.choice((None, 50)), most_keys=rng.choice((1 << 30, 500)))


def test_a_causal_prompt_is_dealt_out_evenly():
    """Row tiles of 1 to 64 KV tiles: the runs differ by little."""
    ctas = _check([8192], [8192], ctas=148, heads=8, group=4, rows=256)
    load = [sum(p[4] + ITEM_TILES for p in pieces) for pieces in ctas]
    assert max(load) <= 1.1 * sum(load) / len(load) + 2 * ITEM_TILES
