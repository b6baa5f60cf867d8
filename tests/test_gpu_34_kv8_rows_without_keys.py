"""GPU tests of query rows that are not finite: NaN where they see a key, and zero with a log-sum-exp of -inf, as any other row, where they see none."""
import math

import pytest
import torch

from pth_flash_attn_b200 import capi
from tests.test_gpu_29_kv8_attention import BF16, F16, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (8, 8, 64), (12, 2, 256)])
@pytest.mark.parametrize("kv,q", [([3, 700, 1], [4, 4, 4]), ([40, 500, 129], [60, 100, 200])])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_rows_that_are_not_finite(kv, q, Hq, Hkv, D, dtype, value):
    """More tokens than keys: the first of them are at negative positions."""
    b = Batch(kv, q, Hq, Hkv, D, dtype, seed=D)
    clean_out, clean_lse = b.attend().out.clone(), b.lse.clone()
    b.check()
    nan = torch.zeros(b.lse.shape, dtype=torch.bool, device="cuda")
    for r, (n, t) in enumerate(zip(kv, q)):
        for i in {0, 1, t // 2, t - 1}:
            token, head = b.starts[r] + i, (5 * i + r) % Hq
            b.q[token, head, 7 * i % D] = value
            nan[token, head] = n - t + i >= 0
    b.out.fill_(7.0)
    b.attend()
    torch.cuda.synchronize()
    assert capi.load_library().device_status() == 0
    assert bool(b.out[nan].isnan().all()) and bool(b.lse[nan].isnan().all())
    assert torch.equal(b.out[~nan], clean_out[~nan]) and torch.equal(b.lse[~nan], clean_lse[~nan])
