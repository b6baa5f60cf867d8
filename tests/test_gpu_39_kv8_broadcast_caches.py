"""GPU tests of caches that are broadcast along a dimension, and of dimensions of one entry with strides of their own."""
import pytest
import torch

from tests.test_gpu_29_kv8_attention import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q", [1, 4, 100])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_heads_that_share_their_cells(D, q):
    """Keys and values of one KV head expanded to four, scales too."""
    b = Batch([700, 130, 1000], [q] * 3, 16, 1, D, seed=D)
    b.k, b.v, b.ks, b.vs = (x.expand(*x.shape[:2], 4, *x.shape[3:]) for x in (b.k, b.v, b.ks, b.vs))
    (b.decode() if q == 1 else b.attend()).check()


@pytest.mark.parametrize("q", [1, 4, 100])
@pytest.mark.parametrize("stride", [0, 16])
def test_one_head_of_any_stride(stride, q):
    b = Batch([700, 130, 1000], [q] * 3, 8, 1, 128, seed=1)
    b.k, b.v = (x.as_strided(x.shape, (x.stride(0), x.stride(1), stride, 1)) for x in (b.k, b.v))
    (b.decode() if q == 1 else b.attend()).check()


@pytest.mark.parametrize("q", [1, 100])
def test_one_page_for_all_blocks(q):
    """A page expanded to many: every block of a table is the same."""
    b = Batch([32], [q] if q == 1 else [32], 8, 2, 128, seed=2, spare=0)
    b.k, b.v, b.ks, b.vs = (x.expand(20, *x.shape[1:]) for x in (b.k, b.v, b.ks, b.vs))
    b.kv_lens = [300]
    b.lens[0] = 300
    b.table = torch.arange(20, dtype=torch.int32)[None]
    b.bt = b.table.cuda()
    (b.decode() if q == 1 else b.attend()).check()
