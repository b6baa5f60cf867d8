"""GPU tests of the 8-bit cache's writer and reader: every cell and scale against a plain form, block of tokens by block."""
import math

import pytest
import torch

from pth_flash_attn_b200 import ops
from tests.kv8_util import E4M3, make_cache, make_table, read_reference, write_reference

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Writes:
    """Requests that hold ``prior`` tokens and get ``new`` ones."""

    def __init__(self, prior, new, Hkv, D, dtype=BF16, *, page=32, group=16, layout="NHD", pad=0, seed=0, strided=False, spread=1.0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.seq = [p + n for p, n in zip(prior, new)]
        self.starts = [0]
        for n in new:
            self.starts.append(self.starts[-1] + n)
        blocks = sum(-(-n // page) for n in self.seq) + 3
        self.table = make_table(self.seq, page, blocks, gen=torch.Generator().manual_seed(seed))
        self.cache = list(make_cache(blocks, page, group, Hkv, D, layout, pad=pad))
        for cells, scale in ((self.cache[0], self.cache[2]), (self.cache[1], self.cache[3])):   # what is held before
            cells.copy_((torch.randn(cells.shape, generator=gen, device="cuda") * 100).clamp(-448, 448))
            scale.copy_(torch.exp2(torch.randint(-12, -5, scale.shape, generator=gen, device="cuda").float()))
        T, extra = self.starts[-1], 3 if strided else 0
        self.key, self.value = ((torch.randn((T, Hkv, D + extra), generator=gen, device="cuda")
                                 * torch.exp(spread * torch.randn((T, Hkv, 1), generator=gen, device="cuda"))).to(dtype)[..., extra:] for _ in range(2))
        self.longest = max(new, default=0)

    def want(self):
        return write_reference(self.key, self.value, *self.cache, self.table, self.seq, self.starts, self.longest)

    def run(self):
        ops.kv8_write(self.key, self.value, *self.cache, self.table.cuda(), _i32(self.seq), _i32(self.starts), self.longest)
        return self

    def check(self):
        want = self.want()
        self.run()
        torch.cuda.synchronize()
        for name, got, w in zip(("k_cache", "v_cache", "k_scale", "v_scale"), self.cache, want):
            if got.dtype == E4M3:
                a, b = got.cpu().float(), w.float()
                same = (a == b) | (a.isnan() & b.isnan())
            else:
                same = (got.cpu() == w) | (got.cpu().isnan() & w.isnan())
            assert bool(same.all()), f"{name}: {int((~same).sum())} differ, first {torch.nonzero(~same)[0].tolist()}"


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_tokens_one_by_one(D, dtype):
    """One token of each request: blocks that begin, go on, and need a larger scale."""
    prior = list(range(0, 40)) + [127, 128, 1000]
    Writes(prior, [1] * len(prior), 2, D, dtype, seed=D, spread=1.5).check()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("page,group", [(16, 16), (32, 32), (48, 48), (64, 16), (816, 48), (816, 816), (128, 64)])
def test_prompts(page, group, dtype):
    Writes([0, 5, 16, 31, 100, 0], [100, 3, 16, 50, 1, 0], 3, 64, dtype, page=page, group=group, seed=page).check()


@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("D", [64, 256])
def test_layouts_and_strides(layout, strided, D):
    Writes([7, 0, 20], [40, 17, 1], 2, D, layout=layout, pad=16, strided=strided, seed=3).check()


def test_many_ragged_requests():
    new = [(7 * i * i + 3 * i) % 23 for i in range(150)]
    prior = [(5 * i) % 37 for i in range(150)]
    Writes(prior, new, 1, 64, seed=5).check()


@pytest.mark.parametrize("group", [16, 64])
def test_special_values(group):
    """Infinities, NaN, zeros, numbers at a power of two's border and at the ends of the range."""
    w = Writes([0, 8, 0, 0, 0, 0], [16, 8, 16, 3, 16, 16], 1, 64, F32, page=64, group=group, seed=1)
    w.key[0:16] = 0.0
    w.key[3, 0, 5] = math.inf
    w.key[4, 0, 6] = -math.inf
    w.key[5, 0, 7] = math.nan
    w.key[16:24] = math.nan
    w.key[24:40] = 448.0 * 2.0 ** 3
    w.value[24:40] = 448.0 * 2.0 ** 3 * (1 + 2.0 ** -23)
    w.key[40:43] = 2.0 ** -140
    w.value[40:43] = torch.finfo(F32).max
    w.key[43:59] = 2.0 ** -130
    w.value[43:59, 0, :32] = 1.5 * 2.0 ** -9 * 2.0 ** -7
    w.check()


def test_scales_that_are_no_numbers_and_of_other_writers():
    w = Writes([3, 5, 9, 12, 15], [1] * 5, 1, 64, F32, page=16, seed=2)
    b = w.table[:, 0].long().cuda()
    w.cache[2][b[0]], w.cache[2][b[1]], w.cache[2][b[2]] = math.nan, -1.0, math.inf
    w.cache[2][b[3]], w.cache[2][b[4]] = 0.3, 3e-5   # (kept, and too small)
    w.key[3] *= 0.01
    # (NaN cells aside: a scale that is no number leaves zeros, whose signs do not matter)
    w.check()


def test_tokens_without_a_place_are_skipped():
    w = Writes([0, 0, 10, 0], [40, 40, 3, 9], 2, 64, page=32, seed=4)
    w.table[0, 1] = -1
    w.table[1, 0] = 1 << 20
    w.seq[2] = 5000              # past the table
    w.seq[3] = 4                 # five tokens at negative positions
    w.longest = 38               # two tokens of the first two requests are past the bound
    w.check()


def test_empty_calls():
    w = Writes([0, 3], [0, 0], 1, 64)
    before = [x.clone() for x in w.cache]
    w.run()
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(torch.uint8) if a.dtype == E4M3 else a, b.view(torch.uint8) if b.dtype == E4M3 else b) for a, b in zip(w.cache, before)
               if not bool(a.float().isnan().any()))


def test_a_write_again_changes_nothing():
    w = Writes([3, 0, 30], [20, 50, 1], 2, 128, seed=6)
    w.run()
    first = [x.clone() for x in w.cache]
    w.run()
    for a, b in zip(w.cache, first):
        assert torch.equal(a.float().nan_to_num(9.0), b.float().nan_to_num(9.0))


def test_appended_tokens_hold_what_a_prompt_would():
    """Token by token, the scale ends where a prompt's is; cells differ by what rounding again costs, a step of e4m3 at most twice."""
    whole = Writes([0], [33], 2, 64, seed=7)
    steps = Writes([0], [33], 2, 64, seed=7)
    whole.run()
    for i in range(33):
        ops.kv8_write(steps.key[i:i + 1], steps.value[i:i + 1], *steps.cache, steps.table.cuda(), _i32([i + 1]), _i32([0, 1]), 1)
    torch.cuda.synchronize()
    b = steps.table[0].long().cuda()
    at = torch.arange(33, device="cuda")
    for cells, scales in ((0, 2), (1, 3)):
        assert torch.equal(whole.cache[scales][b[at // 32], at % 32 // 16], steps.cache[scales][b[at // 32], at % 32 // 16])
        x, y = (w.cache[cells][b[at // 32], at % 32].float() for w in (whole, steps))
        # both round the same quotient, one of them after other roundings at finer steps: each is off by half a step at most
        assert bool(((x - y).abs() <= 2.0 ** -3 * x.abs().clamp(min=2.0 ** -6)).all())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
def test_reads(D, dtype, layout):
    w = Writes([0] * 5, [100, 1, 0, 33, 900], 2, D, seed=D, layout=layout)
    first, rows = [0, 0, 5, 16, 70], [100, 1, 0, 10, 800]
    starts = [0]
    for n in rows:
        starts.append(starts[-1] + n)
    out = [torch.full((starts[-1] + 3, 2, D + 16), 7.0, dtype=dtype, device="cuda")[..., :D] for _ in range(2)]
    want = [read_reference(c, s, w.table, first, starts, 700, o) for c, s, o in ((w.cache[0], w.cache[2], out[0]), (w.cache[1], w.cache[3], out[1]))]
    ops.kv8_read(*out, *w.cache, w.table.cuda(), _i32(first), _i32(starts), 700)
    torch.cuda.synchronize()
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.parametrize("page,group", [(16, 16), (48, 48), (816, 48)])
def test_reads_of_many_requests_and_missing_cells(page, group):
    """Rows enough for CTAs of sixteen; blocks outside the cache, positions past the table and in front of the first."""
    lens = [(13 * i) % 400 for i in range(60)]
    w = Writes([0] * 60, lens, 1, 64, page=page, group=group, seed=1)
    w.table[7, 0] = -1
    w.table[9, 0] = 1 << 25
    first = [0] * 60
    first[3], first[4] = -5, 100000
    want = [read_reference(c, s, w.table, first, w.starts, 1000, torch.zeros_like(w.key)) for c, s in ((w.cache[0], w.cache[2]), (w.cache[1], w.cache[3]))]
    out = [torch.full_like(w.key, 3.0) for _ in range(2)]
    ops.kv8_read(*out, *w.cache, w.table.cuda(), _i32(first), _i32(w.starts), 1000)
    torch.cuda.synchronize()
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_round_trip_error():
    """What was written comes back within half a step of e4m3: 2^-4 of the value, or 2^-10 of the scale."""
    w = Writes([0, 0], [200, 77], 4, 128, seed=9)
    w.run()
    out = [torch.empty_like(w.key) for _ in range(2)]
    ops.kv8_read(*out, *w.cache, w.table.cuda(), _i32([0, 0]), _i32(w.starts), 200)
    for got, x in zip(out, (w.key, w.value)):
        most = x.float().abs().amax()
        assert bool(((got.float() - x.float()).abs() <= 2.0 ** -4 * x.float().abs() + 2.0 ** -10 * most / 224).all())


def test_reads_with_many_requests_without_rows_between():
    """Requests of no rows, thousands of them between two that have some."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    page, Hkv, D, R = 32, 2, 64, 9000
    cache = make_cache(40, page, 16, Hkv, D)
    for cells, scale in ((cache[0], cache[2]), (cache[1], cache[3])):
        cells.copy_((torch.randn(cells.shape, generator=gen, device="cuda") * 100).clamp(-448, 448))
        scale.copy_(torch.exp2(torch.randint(-12, -5, scale.shape, generator=gen, device="cuda").float()))
    rows = [0] * R
    for r, n in ((3, 5), (4, 1), (17, 40), (4099, 2), (8000, 1), (8001, 33), (8999, 7)):
        rows[r] = n
    starts = [0]
    for n in rows:
        starts.append(starts[-1] + n)
    table = torch.randint(0, 40, (R, 2), generator=torch.Generator().manual_seed(7), dtype=torch.int32)
    first = [r % 11 for r in range(R)]
    out = [torch.full((starts[-1], Hkv, D), 7.0, dtype=BF16, device="cuda") for _ in range(2)]
    want = [read_reference(c, s, table, first, starts, 40, o) for c, s, o in ((cache[0], cache[2], out[0]), (cache[1], cache[3], out[1]))]
    ops.kv8_read(*out, *cache, table.cuda(), _i32(first), _i32(starts), 40)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
