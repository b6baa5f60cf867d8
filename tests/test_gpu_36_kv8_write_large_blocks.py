"""GPU tests of single tokens written to blocks of many tokens: the older ones, up to 815 of them, are rounded again where the token needs a larger scale."""
import pytest
import torch

from tests.test_gpu_30_kv8_write_read import BF16, F16, F32, Writes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page,group", [(48, 48), (64, 64), (128, 128), (816, 816), (816, 272)])
def test_single_tokens(page, group, D, dtype):
    """Offsets about a warp's 32 rows and the block's ends; larger tokens, smaller ones, and some of each beside one another."""
    prior = [0, 1, 31, 32, 33, 34, group // 2, group - 2, group - 1, group, group + 1, group + 33, 2 * group - 1]
    w = Writes(prior, [1] * len(prior), 3, D, dtype, page=page, group=group, seed=D + group, spread=2.0)
    w.check()


@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("size", [2.0 ** -9, 2.0 ** 9])
def test_all_of_them_grow_or_none(layout, size):
    prior = [815 - 13 * i for i in range(60)]
    w = Writes(prior, [1] * 60, 2, 128, BF16, page=816, group=816, layout=layout, pad=16, seed=1)
    w.key *= size
    w.value *= size
    w.check()


def test_a_few_tokens_and_single_ones_give_the_same():
    """The call of one token of each request, and one that may have more, take kernels of their own."""
    one = Writes([700, 33, 815, 64], [1] * 4, 2, 64, page=816, group=816, seed=3, spread=2.0).run()
    two = Writes([700, 33, 815, 64], [1] * 4, 2, 64, page=816, group=816, seed=3, spread=2.0)
    two.longest = 4
    two.run()
    for a, b in zip(one.cache, two.cache):
        assert torch.equal(a.float().nan_to_num(9.0), b.float().nan_to_num(9.0))


def test_scales_that_are_no_numbers_in_front_of_many_older_tokens():
    w = Writes([500, 700, 40], [1] * 3, 1, 64, F32, page=816, group=816, seed=2)
    b = w.table[:, 0].long().cuda()
    w.cache[2][b[0]], w.cache[2][b[1]], w.cache[3][b[2]] = float("nan"), -1.0, float("inf")
    w.check()
