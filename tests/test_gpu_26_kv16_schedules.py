"""GPU tests of the schedules of attention over the 16-bit cache that small batches do not reach: prompts in waves of items (several
waves, CTAs without a share of the rest), more requests than a plan holds, requests of many tokens without states, boxes past
32-bit offsets."""
import math

import pytest
import torch

from pth_flash_attn_b200 import capi, ops
from tests.kv16_plan import Plan
from tests.kv16_util import check, reference
from tests.test_gpu_20_kv16_attention import BF16, F16, Batch, _workspace

pytestmark = pytest.mark.gpu


def _sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def _ragged(seed, count, lo, hi):
    return torch.randint(lo, hi + 1, (count,), generator=torch.Generator().manual_seed(seed)).tolist()


def _twice(b):
    """The same workspace again: its counters were left at zero, and the bits do not depend on who arrives last."""
    b.cross().check()
    first = b.out.clone()
    b.out.fill_(math.nan)
    b.cross()
    torch.cuda.synchronize()
    live = ~torch.isnan(first)
    assert torch.equal(b.out[live], first[live]) and bool(live.all())


# head counts, head size, requests, their tokens, their states at most; states of every eighth request; of the last sixth, at most
WAVES = [
    (8, 8, 128, 75, (100, 256), 300, 6000, 2500),
    (16, 8, 128, 70, (60, 300), 300, 5000, 2500),
    (32, 4, 128, 60, (1, 200), 500, 6000, 3000),
    (4, 4, 256, 130, (90, 128), 300, 5000, 2500),
    (16, 2, 256, 70, (10, 100), 500, 5000, 3000),
    (8, 8, 64, 140, (30, 128), 400, 8000, 4000),
    (16, 4, 64, 90, (1, 130), 700, 9000, 4000),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("Hq,Hkv,D,requests,tokens,few,many,tail", WAVES)
def test_waves_of_items(Hq, Hkv, D, requests, tokens, few, many, tail, dtype):
    """Some CTAs' waves hold items of far longer requests: they get no share of the rest, and pieces of a divided item lie on both sides
    of them."""
    q_lens, kv_lens = _ragged(1, requests, *tokens), _ragged(2, requests, 1, few)
    kv_lens[3::8] = [many] * len(kv_lens[3::8])
    kv_lens[-(requests // 6):] = _ragged(3, requests // 6, tail // 2, tail)
    plan = Plan(kv_lens, q_lens, Hq, Hkv, D, _sms())
    assert plan.waves >= 2 and 0 in plan.shares and plan.skipped > 0
    _twice(Batch(kv_lens, q_lens, Hq, Hkv, D, dtype, seed=D))


@pytest.mark.parametrize("Hq,Hkv,D,requests", [(8, 8, 128, 150), (8, 4, 256, 200), (16, 16, 64, 130)])
def test_many_waves_with_empty_requests(Hq, Hkv, D, requests):
    q_lens, kv_lens = _ragged(3, requests, 0, 300), _ragged(4, requests, 0, 700)
    q_lens[::7] = [0] * len(q_lens[::7])
    kv_lens[1::7] = [0] * len(kv_lens[1::7])
    plan = Plan(kv_lens, q_lens, Hq, Hkv, D, _sms())
    assert plan.waves >= 4
    _twice(Batch(kv_lens, q_lens, Hq, Hkv, D, BF16, seed=D))


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 8, 128), (8, 8, 64), (4, 4, 256)])
def test_waves_over_pages_without_boxes(Hq, Hkv, D):
    q_lens, kv_lens = _ragged(5, 150, 60, 200), _ragged(6, 150, 1, 500)
    assert Plan(kv_lens, q_lens, Hq, Hkv, D, _sms()).waves >= 1
    _twice(Batch(kv_lens, q_lens, Hq, Hkv, D, BF16, page=5, seed=D))


@pytest.mark.parametrize("requests", [4096, 4097, 6000])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 64), (2, 2, 128), (2, 1, 256)])
def test_requests_that_a_plan_does_not_hold(Hq, Hkv, D, requests):
    """Up to 4,096 go out in waves, more of them in equal runs."""
    q_lens, kv_lens = _ragged(7, requests, 0, 2), _ragged(8, requests, 0, 60)
    q_lens[100], kv_lens[100] = 300, 5000
    q_lens[-1], kv_lens[-1] = 40, 1
    plan = Plan(kv_lens, q_lens, Hq, Hkv, D, _sms())
    assert (plan.waves > 0) == (requests <= 4096)
    _twice(Batch(kv_lens, q_lens, Hq, Hkv, D, BF16, seed=requests, page=64))


@pytest.mark.parametrize("requests", [1000, 5000])
def test_decode_of_many_requests(requests):
    kv_lens = _ragged(9, requests, 0, 90)
    kv_lens[requests // 2] = 30000
    Batch(kv_lens, [1] * requests, 8, 2, 64, BF16, seed=requests, page=64).decode().check()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kv_lens,q_lens", [([500, 0, 300, 0], [300, 2048, 100, 1500]), ([0, 0], [1000, 1]), ([0], [2048]), ([0, 9000, 0], [3, 5, 700])])
def test_many_tokens_without_states(kv_lens, q_lens, D):
    _twice(Batch(kv_lens, q_lens, 8, 2, D, BF16, seed=31))


@pytest.mark.parametrize("layout", ["NHD", "HND"])
def test_boxes_past_32_bit_offsets(layout):
    """A cache of 5 GB whose used pages lie at its end, read by tokens enough for the prompts' kernel."""
    Hkv, D, page, kv_lens, q_lens = 8, 128, 16, [500, 77, 2000], [100, 300, 20]
    blocks = (5 << 30) // (page * Hkv * D * 2)
    shape = (2, blocks, page, Hkv, D) if layout == "NHD" else (2, blocks, Hkv, page, D)
    storage = torch.empty(shape, dtype=BF16, device="cuda")
    pages = [-(-n // page) for n in kv_lens]
    table = torch.zeros((3, max(pages)), dtype=torch.int32)
    last = blocks
    for r, n in enumerate(pages):
        table[r, :n] = torch.arange(last - n, last, dtype=torch.int32)
        last -= n
    storage[:, last:].normal_()
    k, v = storage if layout == "NHD" else storage.transpose(2, 3)
    starts = [0, 100, 400, 420]
    q = torch.randn((420, 32, D), device="cuda").to(BF16)
    out, lse = torch.empty_like(q), torch.empty((420, 32), device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    ops.kv16_cross_attention(out, lse, q, k, v, table.cuda(), torch.tensor(kv_lens, **i32), torch.tensor(starts, **i32), 300, D ** -0.5, _workspace(D))
    check(out, lse, reference(q, k, v, table, kv_lens, starts, D ** -0.5))
    assert capi.load_library().device_status() == 0
