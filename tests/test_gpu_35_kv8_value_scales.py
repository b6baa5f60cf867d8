"""GPU tests of the scales of values: one that is no power of two costs nothing, and one that a token does not see changes nothing for it."""
import math

import pytest
import torch

from pth_flash_attn_b200 import capi
from tests.kv8_util import E4M3, check
from tests.test_gpu_29_kv8_attention import BF16, F16, Batch

pytestmark = pytest.mark.gpu


def _half_step(x, bits):
    """Half the distance of neighbouring numbers of `bits` bits at x."""
    return torch.exp2(torch.floor(torch.log2(x.abs())) - bits)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("scale", [1 + 2.0 ** -11, 0.013, 0.7 + 2.0 ** -12, 1.4985])
def test_prompts_over_one_scale_that_is_no_power_of_two(D, scale):
    """Equal weights over equal values: nothing is rounded but the result (and 32-bit sums, exponentials and a quotient, 2^-20 of it together)."""
    b = Batch([700, 90], [90, 90], 8, 2, D, F16, seed=D)
    b.q.zero_()
    b.vs = torch.full((1, 1, 1), scale, device="cuda").expand(b.vs.shape)
    b.ks = torch.full((1, 1, 1), 2.0 ** -7, device="cuda").expand(b.ks.shape)
    value = (1.0 + torch.arange(D, device="cuda") % 8 / 8) * torch.exp2((torch.arange(D, device="cuda") % 5).float())   # (e4m3 numbers)
    for r, n in enumerate(b.kv_lens):
        at = torch.arange(n, device="cuda")
        b.v[b.bt[r].long()[at // b.page], at % b.page] = value.to(E4M3)
    b.attend()
    want = (value.double() * float(torch.tensor(scale))).expand(b.out.shape)
    assert bool(((b.out.double() - want).abs() <= _half_step(want, 11) + 2.0 ** -20 * want).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (16, 16, 64), (12, 2, 256)])
@pytest.mark.parametrize("up", [2.0 ** 10, 2.0 ** 16, 2.0 ** 30, 2.0 ** 60])
def test_prompts_with_a_larger_scale_under_keys_that_some_tokens_do_not_see(Hq, Hkv, D, dtype, up):
    """The last block of a request's own tokens: those in front of it get the same bits, those that see it what the formula says."""
    kv, q = [1024, 256, 3000], [100, 256, 64]
    b = Batch(kv, q, Hq, Hkv, D, dtype, seed=D)
    clean = b.attend().out.clone(), b.lse.clone()
    seen = torch.zeros(b.out.shape[0], dtype=torch.bool, device="cuda")
    for r, n in enumerate(kv):
        first = (n - 20) // 16 * 16
        b.vs[int(b.table[r, first // b.page]), first % b.page // 16] *= up * (1.0 if dtype == BF16 else 2.0 ** -6)
        seen[b.starts[r] + first - (n - q[r]):b.starts[r + 1]] = True
    b.out.fill_(math.nan)
    b.attend()
    torch.cuda.synchronize()
    assert capi.load_library().device_status() == 0
    assert torch.equal(b.out[~seen], clean[0][~seen]) and torch.equal(b.lse[~seen], clean[1][~seen])
    if dtype == BF16 or up <= 2.0 ** 16:   # (fp16 has no larger results)
        want = b.reference()
        check(b.out[seen], b.lse[seen], tuple(x[seen] for x in want))
