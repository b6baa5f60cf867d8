"""GPU tests of NaN among the cached values where the kernel of few rows computes several tokens of a request: long caches, and prompts over broadcast cells,
whose row tiles it takes one by one."""
import math

import pytest
import torch

from pth_flash_attn_b200 import capi
from tests.test_gpu_29_kv8_attention import Batch, _sees

pytestmark = pytest.mark.gpu


def _check(b, q, cells, window, causal):
    """`cells`: (request, key, dimension or None for all) that become NaN, in all heads."""
    clean = b.attend(window, causal).out.clone(), b.lse.clone()
    nan = torch.zeros_like(b.out, dtype=torch.bool)
    for r, key, d in cells:
        where = slice(None) if d is None else d
        b.v[int(b.table[r, key // b.page]), key % b.page, :, where] = math.nan
        for i in range(q[r]):
            if _sees(b, r, i, key, window, causal):
                nan[b.starts[r] + i, :, where] = True
    b.out.fill_(7.0)
    b.attend(window, causal)
    torch.cuda.synchronize()
    assert capi.load_library().device_status() == 0
    assert torch.equal(b.out.isnan(), nan) and torch.equal(b.out[~nan], clean[0][~nan]) and torch.equal(b.lse, clean[1])


@pytest.mark.parametrize("Hq,Hkv,D,q", [(8, 2, 128, 2), (8, 2, 128, 4), (8, 2, 128, 8), (8, 8, 64, 16), (32, 32, 128, 32), (12, 2, 256, 4)])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 3), (True, 500), (False, 200)])
def test_long_caches(Hq, Hkv, D, q, causal, window):
    kv = [50000, 3000, 140, 129, 20]
    b = Batch(kv, [q] * 5, Hq, Hkv, D, seed=D + q, page=64)
    cells = []
    for r, n in enumerate(kv):
        cells += [(r, n - 1, 3), (r, n - min(q, n) // 2, D - 1), (r, max(0, n - q - 1), 5), (r, max(0, n - 1 - window), None), (r, max(0, n - q - window + 1), 9), (r, n // 2, 11)]
    _check(b, [q] * 5, cells, window, causal)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 100), (False, 150)])
def test_prompts_over_broadcast_cells(D, causal, window):
    q = [300, 130, 64]
    b = Batch([700, 130, 1000], q, 8, 1, D, seed=D, page=64)
    b.k, b.v, b.ks, b.vs = (x.expand(*x.shape[:2], 2, *x.shape[3:]) for x in (b.k, b.v, b.ks, b.vs))
    cells = [(0, 699, 1), (0, 500, None), (0, 410, 2), (0, 300, 3), (1, 129, 4), (1, 1, 5), (2, 950, 6), (2, 900, 7)]
    _check(b, q, cells, window, causal)
