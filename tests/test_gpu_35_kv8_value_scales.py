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


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("Hq,Hkv,D,q", [(8, 2, 128, 4), (8, 2, 128, 2), (8, 2, 128, 8), (8, 8, 64, 4), (12, 2, 256, 4)])
@pytest.mark.parametrize("up", [2.0 ** 10, 2.0 ** 16, 2.0 ** 30, 2.0 ** 60])
def test_few_tokens_with_a_larger_scale_under_keys_that_some_do_not_see(Hq, Hkv, D, q, dtype, up):
    """A block that begins with the last token but one: those in front of it are as exact as without it."""
    kv = [1026, 258, 5010, 18, 130]
    b = Batch(kv, [q] * len(kv), Hq, Hkv, D, dtype, seed=D + q)
    clean = b.reference()
    seen = torch.zeros(b.out.shape[0], dtype=torch.bool, device="cuda")
    for r, n in enumerate(kv):
        first = n - 2
        b.vs[int(b.table[r, first // b.page]), first % b.page // 16] *= up * (1.0 if dtype == BF16 else 2.0 ** -6)
        seen[b.starts[r + 1] - 2:b.starts[r + 1]] = True
    b.attend()
    torch.cuda.synchronize()
    assert capi.load_library().device_status() == 0
    check(b.out[~seen], b.lse[~seen], tuple(x[~seen] for x in clean))
    if dtype == BF16 or up <= 2.0 ** 16:
        want = b.reference()
        check(b.out[seen], b.lse[seen], tuple(x[seen] for x in want))


@pytest.mark.parametrize("first", [0.0, 2.0 ** -126, 2.0 ** -60, 2.0 ** 60])
def test_scales_of_the_first_keys_far_from_the_others(first):
    """A whole tile of values of no size, or of a size of their own, in front of the others."""
    for q in (1, 4, 100):
        b = Batch([1000, 140, 300], [q] * 3, 8, 2, 128, seed=5)
        for r in range(3):
            blocks = b.bt[r, :4].long()   # (128 keys)
            b.vs[blocks] = first
            if first <= 2.0 ** -126:
                b.v[blocks] = 0.0
        (b.decode() if q == 1 else b.attend()).check()


@pytest.mark.parametrize("q", [1, 4])
def test_a_row_whose_weight_lies_under_small_scales(q):
    """Scales of 2^-24 of the others', under the keys that have nearly all of the weight: bits of their own."""
    b = Batch([900], [q], 8, 2, 128, seed=6, scales=(-7, -6))
    at = torch.arange(600, 616, device="cuda")
    where = b.bt[0].long()[at // b.page], at % b.page
    b.q[...] = b.q.abs()
    b.k[where] = torch.full((16, 2, 128), 448.0, device="cuda").to(E4M3)   # scores far above the others'
    b.vs[b.bt[0, 600 // b.page].long(), 600 % b.page // 16] *= 2.0 ** -24
    want = b.reference()
    (b.decode() if q == 1 else b.attend())
    torch.cuda.synchronize()
    # what the other keys weigh is less than 2^-60 of it, so nothing but 16 weights of 2^-11 each and the result is rounded
    spread = torch.einsum("jhd->hd", b.v[where].double().abs()).repeat_interleave(4, 0) * 2.0 ** -31 / 16
    assert bool(((b.out.double() - want[0]).abs() <= 2.0 ** -8 * want[0].abs() + 2.0 ** -10 * 16 * spread).all())
