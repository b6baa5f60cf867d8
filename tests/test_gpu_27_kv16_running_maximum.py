"""GPU tests of the running bound of a row's scores in attention over the 16-bit cache, at every head size and in both kernels: keys
that outgrow what came before, one after another, in every part of a step and of a piece; scores that rise, fall, or go far past 1."""
import math

import pytest
import torch

from tests.kv16_util import check, reference
from tests.test_gpu_20_kv16_attention import BF16, F16, Batch

pytestmark = pytest.mark.gpu
HEADS = [(8, 2, 64), (8, 2, 128), (8, 2, 256), (16, 1, 128), (32, 1, 64), (32, 1, 256)]


def _scores(b, r, scores):
    """Keys of request r whose product with a row of ones, scaled, is `scores`; a row's queries are a factor of ones, of either sign."""
    at = torch.arange(b.kv_lens[r])
    b.k[b.table[r].long()[at // b.page].cuda(), (at % b.page).cuda()] = (scores / b.D ** 0.5)[:, None, None].to(b.k.dtype).expand(-1, *b.k.shape[2:]).cuda()
    t0, t1 = b.starts[r], b.starts[r + 1]
    factor = 1 - 1.75 * torch.rand((t1 - t0, b.Hq), generator=torch.Generator().manual_seed(r))
    factor[0] = 1
    b.q[t0:t1] = factor[..., None].to(b.q.dtype).expand(-1, -1, b.D).cuda()


# Where a key outgrows all before it, by 12 (2^17): in either half of the first 128 keys and of later ones, at edges of steps and
# tiles, in neighbours, far behind.
PEAKS = [[70], [63, 64], [127, 128], [5, 70, 130, 200, 260, 330], [200, 300], [191, 192, 193], [64, 128, 192, 256, 320, 384], [999], [0, 1, 2, 3],
         [100, 400, 700, 990]]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("peaks", PEAKS)
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("q_lens", [[1, 1], [90, 1]])
def test_keys_that_outgrow_what_came_before(q_lens, Hq, Hkv, D, peaks, dtype):
    b = Batch([1000, 40], q_lens, Hq, Hkv, D, dtype, seed=40)
    scores = torch.randn(1000, generator=torch.Generator().manual_seed(41)) * 0.5
    for i, at in enumerate(peaks):
        scores[at] = 12.0 * (i + 1)
    _scores(b, 0, scores)
    if max(q_lens) == 1:
        b.decode().check(what=str(peaks))
        b.out.fill_(math.nan)
    b.cross().check(what=str(peaks))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("slope", [0.02, -0.02, 0.3, -0.3])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("q_lens", [[1, 1], [90, 1]])
@pytest.mark.parametrize("n", [333, 20000])
def test_scores_that_rise_or_fall(n, q_lens, Hq, Hkv, D, slope, dtype):
    """Key by key, with steps back between: the bound moves again and again, and pieces of a request have bounds of their own."""
    b = Batch([n, 40], q_lens, Hq, Hkv, D, dtype, seed=42)
    _scores(b, 0, torch.arange(n) * slope * min(1.0, 1000 / n) + torch.randn(n, generator=torch.Generator().manual_seed(43)))
    if max(q_lens) == 1:
        b.decode().check(what=str(slope))
        b.out.fill_(math.nan)
    b.cross().check(what=str(slope))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("q_lens", [[1] * 4, [70, 200, 130, 257]])
def test_large_scores(q_lens, Hq, Hkv, D, dtype):
    b = Batch([700, 128, 1, 3000], q_lens, Hq, Hkv, D, dtype, scale_up=30.0, seed=5)
    if max(q_lens) == 1:
        b.decode().check()
        b.out.fill_(math.nan)
    b.cross().check()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_cross_infinite_query_makes_its_row_nan_and_no_other(D):
    b = Batch([300, 300], [40, 90], 8, 2, D, BF16, seed=8)
    b.q[7, 3] = math.inf
    b.cross()
    torch.cuda.synchronize()
    assert bool(torch.isnan(b.out[7, 3]).all())
    keep = torch.ones(130, 8, dtype=torch.bool, device="cuda")
    keep[7, 3] = False
    q = b.q.clone()
    q[7, 3] = 0
    want = reference(q, b.k, b.v, b.table, b.kv_lens, b.starts, D ** -0.5)
    check(b.out[keep][None], b.lse[keep][None], [w[keep][None] for w in want])
