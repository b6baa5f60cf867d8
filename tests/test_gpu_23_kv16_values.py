"""GPU tests of attention over the 16-bit cache at values from the ends of its types: infinities among the visible values, values
near the largest of bf16, and far below one."""
import math

import pytest
import torch

from pth_flash_attn_b200 import ops
from tests.kv16_util import check, reference
from tests.test_gpu_20_kv16_attention import BF16, EDGES, F16, Q_LENS, STATES, Batch

pytestmark = pytest.mark.gpu


def _where(b, r, at):
    """Block and slot of request r's keys `at`."""
    at = torch.as_tensor(at)
    return b.table[r].long()[at // b.page].cuda(), (at % b.page).cuda()


def _check_with_infinities(b, what=""):
    """Columns without an infinite value as always; the others are what the sum of positive weights times values is."""
    torch.cuda.synchronize()
    v = b.v.clone()
    v[~torch.isfinite(v)] = 0   # (what no request sees is NaN: the reference does not see it either)
    want = reference(b.q, b.k, v, b.table, b.kv_lens, b.starts, b.D ** -0.5)
    out, G = b.out.clone(), b.Hq // b.k.shape[2]
    for r, n in enumerate(b.kv_lens):
        t0, t1 = b.starts[r], b.starts[r + 1]
        if n == 0 or t1 == t0:
            continue
        seen = b.v[_where(b, r, torch.arange(n))]
        plus, minus = ((seen == x).any(0).repeat_interleave(G, 0)[None].expand(t1 - t0, -1, -1) for x in (math.inf, -math.inf))
        rows = out[t0:t1]
        assert bool((rows[plus & ~minus] == math.inf).all()), f"{what}: request {r}, +inf"
        assert bool((rows[minus & ~plus] == -math.inf).all()), f"{what}: request {r}, -inf"
        assert bool(torch.isnan(rows[plus & minus]).all()), f"{what}: request {r}, both"
        rows[plus | minus] = want[0][t0:t1][plus | minus].to(out.dtype)
    check(out, b.lse, want, what)


def _plant(b, seed=0):
    """Infinities at one key of every request, and both signs at two keys, each in columns of its own."""
    gen = torch.Generator().manual_seed(seed)
    for r, n in enumerate(b.kv_lens):
        if n == 0:
            continue
        for column, sign in ((3, 1), (17, -1), (40, 1), (41, -1), (b.D - 1, 1)):
            block, slot = _where(b, r, int(torch.randint(n, (), generator=gen)))
            b.v[block, slot, :, column] = sign * math.inf
        if n > 1:
            for at, sign in ((0, 1), (n - 1, -1)):
                block, slot = _where(b, r, at)
                b.v[block, slot, :, 7] = sign * math.inf
    return b


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 64), (8, 2, 128), (6, 1, 256), (32, 2, 128), (64, 2, 64), (32, 1, 256), (32, 1, 64)])
@pytest.mark.parametrize("kv_lens", [EDGES, [40000, 3, 777], [2, 5, 9, 33] * 40])
def test_decode_infinite_values(kv_lens, Hq, Hkv, D, dtype):
    _check_with_infinities(_plant(Batch(kv_lens, [1] * len(kv_lens), Hq, Hkv, D, dtype, seed=D + Hq)).decode())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("q_lens", [[1] * 12, [3] * 12, Q_LENS])
def test_cross_infinite_values(q_lens, D, dtype):
    _check_with_infinities(_plant(Batch(STATES, q_lens, 8, 2, D, dtype, seed=D)).cross())
    _check_with_infinities(_plant(Batch([30000, 500], q_lens[-2:], 8, 2, D, dtype, seed=D + 1)).cross())


def _stairs(b, r, levels):
    """Keys of request r whose score with queries of ones is `levels`, tile by tile (natural units)."""
    at = torch.arange(b.kv_lens[r])
    score = torch.tensor(levels)[(at * len(levels)) // b.kv_lens[r]]
    b.q[b.starts[r]:b.starts[r + 1]] = 1
    b.k[_where(b, r, at)] = (score / b.D ** 0.5)[:, None, None].to(b.k.dtype).expand(-1, *b.k.shape[2:]).cuda()


# Beside scores that much larger an infinite value's weight is above zero still, if only in more exponents than 32 bits have.
@pytest.mark.parametrize("levels", [(0.0, 30.0), (0.0, 200.0), (0.0, 96.0, 192.0), (0.0, -8.0), (0.0, -200.0)])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [384, 1000, 30000])
def test_decode_infinite_values_of_small_weight(n, D, dtype, levels):
    b = Batch([n, 40], [1, 1], 8, 2, D, dtype, seed=3)
    _stairs(b, 0, levels)
    first, last = _where(b, 0, 5), _where(b, 0, n - 2)
    b.v[(*first, slice(None), 9)] = math.inf
    b.v[(*last, slice(None), 11)] = -math.inf
    _check_with_infinities(b.decode(), str(levels))


# (prompts keep one 16-bit weight a key: there a falling step stays within fp16's numbers, 2^-31 of the largest)
@pytest.mark.parametrize("levels", [(0.0, 30.0), (0.0, 200.0), (0.0, 96.0, 192.0), (0.0, -8.0)])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [384, 1000, 30000])
def test_cross_infinite_values_of_small_weight(n, D, dtype, levels):
    b = Batch([n, 40], [70, 1], 8, 2, D, dtype, seed=3)
    _stairs(b, 0, levels)
    first, last = _where(b, 0, 5), _where(b, 0, n - 2)
    b.v[(*first, slice(None), 9)] = math.inf
    b.v[(*last, slice(None), 11)] = -math.inf
    _check_with_infinities(b.cross(), str(levels))


def test_a_value_that_fp16_cannot_hold():
    """The writer rounds it to infinity; attention over it is infinite, not NaN, whatever its weight's bits are."""
    b = Batch([300] * 64, [1] * 64, 8, 2, 128, F16, seed=4)
    key = torch.randn((64, 2, 128), device="cuda")
    value = torch.randn((64, 2, 128), device="cuda")
    value[:, :, 5], value[:, :, 6] = 70000.0, -1e30
    slots = torch.tensor([int(b.table[r, 250 // 16]) * 16 + 250 % 16 for r in range(64)], device="cuda")
    ops.kv16_write(key, value, b.k, b.v, slots)
    _check_with_infinities(b.decode())
    assert bool((b.out[..., 5] == math.inf).all()) and bool((b.out[..., 6] == -math.inf).all())


def _scale_values(b, size, seed=0):
    """Values of +-size / 2 .. size: of one sign in even columns, of both in odd ones."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.rand(b.v.shape, generator=gen, device="cuda", dtype=torch.float64) / 2 + 0.5) * size
    sign = torch.where(torch.rand(b.v.shape, generator=gen, device="cuda") < 0.5, -1.0, 1.0)
    sign[..., ::2] = 1
    b.v.copy_(torch.where(torch.isnan(b.v), math.nan, x * sign))
    return b


# (bf16 ends at 3.39e38, as 32 bits do: neither sums of weighted values nor their merges may pass it where the result does not)
SIZES = [3.3e38, 1e37, 1e30, 1e-25]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 64), (8, 2, 128), (6, 1, 256), (32, 2, 128), (32, 1, 64), (32, 1, 256)])
def test_decode_values_of_any_size(Hq, Hkv, D, size):
    kv_lens = [1, 2, 0, 129, 700, 5000, 40000]
    _scale_values(Batch(kv_lens, [1] * len(kv_lens), Hq, Hkv, D, BF16, seed=D), size).decode().check()


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("q_lens", [[1] * 6, [3] * 6, [70, 1, 300, 128, 5, 200]])
def test_cross_values_of_any_size(q_lens, D, size):
    _scale_values(Batch([1, 2, 129, 700, 5000, 30000], q_lens, 8, 2, D, BF16, seed=D), size).cross().check()


# Weights that grow behind the first keys, by less than what moves a row's reference and by more.
@pytest.mark.parametrize("levels", [(0.0,), (0.0,) + (5.4,) * 20, (0.0, 5.4, 5.6, 11.2), (0.0, 20.0, 40.0, 60.0)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("q_lens", [[1, 1], [70, 1]])
def test_largest_values_under_growing_weights(q_lens, D, levels):
    b = _scale_values(Batch([5000, 40], q_lens, 8, 2, D, BF16, seed=3), 3.3e38)
    _stairs(b, 0, levels)
    if max(q_lens) == 1:
        b.decode().check(what=str(levels))
    b.cross().check(what=str(levels))
