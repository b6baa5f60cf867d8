"""GPU tests of NaN among the cached keys and values of long prompts: it reaches the tokens that see it, and no other, and no wait of the launch
runs out over it, however long the request."""
import math

import pytest
import torch

from pth_flash_attn_b200 import capi
from tests.test_gpu_29_kv8_attention import Batch, _sees

pytestmark = pytest.mark.gpu

# one long request among others of some pieces for every CTA
KV, Q = [20000] + [1500 + 37 * i for i in range(40)] + [30000], [64] * 41 + [150]


def _plant(b, r, key, what):
    block, slot = int(b.table[r, key // b.page]), key % b.page
    if "k" in what:
        b.k[block, slot] = math.nan
    if "v" in what:
        b.v[block, slot] = math.nan


@pytest.mark.parametrize("D,Hq,Hkv", [(64, 8, 2), (128, 8, 2), (256, 8, 2), (128, 4, 4)])
@pytest.mark.parametrize("window", [0, 5000])
@pytest.mark.parametrize("what", ["own", "all own", "seen", "edge"])
def test_whole_tokens_that_are_nan(D, Hq, Hkv, window, what):
    """A token's keys and values, of all heads: one of the request's own, all of them, one that all see, one at the window's edge."""
    b = Batch(KV, Q, Hq, Hkv, D, seed=D, page=64)
    clean_out, clean_lse = b.attend(window).out.clone(), b.lse.clone()
    keys = []   # (request, key, of what)
    for r in (0, 7, 41):
        n, t = KV[r], Q[r]
        if what == "own":
            keys.append((r, n - 20, "kv"))
        elif what == "all own":
            keys += [(r, key, "v") for key in range(n - t + 1, n)]
        elif what == "seen":
            keys.append((r, n - 1000, "v"))
        else:
            keys.append((r, max(0, n - t + 10 - window) if window else 3, "v"))
    nan_out, nan_lse = torch.zeros_like(b.out, dtype=torch.bool), torch.zeros_like(b.lse, dtype=torch.bool)
    for r, key, of in keys:
        _plant(b, r, key, of)
        for i in range(Q[r]):
            if _sees(b, r, i, key, window, True):
                nan_out[b.starts[r] + i] = True
                nan_lse[b.starts[r] + i] |= "k" in of
    b.out.fill_(7.0)
    b.attend(window)
    torch.cuda.synchronize()
    assert capi.load_library().device_status() == 0
    assert not bool(b.ws[:4096].any()), "arrival counters are left at zero"
    assert torch.equal(b.out.isnan(), nan_out) and torch.equal(b.lse.isnan(), nan_lse)
    assert torch.equal(b.out[~nan_out], clean_out[~nan_out]) and torch.equal(b.lse[~nan_lse], clean_lse[~nan_lse])


@pytest.mark.parametrize("D", [64, 128, 256])
def test_some_dimensions_and_scales(D):
    """NaN in a few dimensions of many own tokens, and in the scale of a block of them."""
    b = Batch([20000, 700, 9000], [256, 200, 300], 8, 2, D, seed=D, page=64)
    clean = b.attend().out.clone()
    gen = torch.Generator().manual_seed(D)
    nan = torch.zeros_like(b.out, dtype=torch.bool)
    for r, (n, t) in enumerate(zip(b.kv_lens, [256, 200, 300])):
        for _ in range(60):
            key, h, d = n - 1 - int(torch.randint(t, (1,), generator=gen)), int(torch.randint(2, (1,), generator=gen)), int(torch.randint(D, (1,), generator=gen))
            b.v[int(b.table[r, key // b.page]), key % b.page, h, d] = math.nan
            nan[b.starts[r] + key - (n - t):b.starts[r + 1], h * 4:(h + 1) * 4, d] = True
        key = (n - t // 2) // 16 * 16
        b.vs[int(b.table[r, key // b.page]), key % b.page // 16, 1] = math.nan
        nan[b.starts[r] + key - (n - t):b.starts[r + 1], 4:] = True
    b.attend()
    torch.cuda.synchronize()
    assert capi.load_library().device_status() == 0
    assert torch.equal(b.out.isnan(), nan) and torch.equal(b.out[~nan], clean[~nan])
