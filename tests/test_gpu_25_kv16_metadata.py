"""GPU tests of attention over the 16-bit cache with start offsets that no scheduler would write: nothing outside the tensors is touched."""
import pytest
import torch

from pth_flash_attn_b200 import capi
from tests.kv16_util import check, reference
from tests.test_gpu_20_kv16_attention import BF16, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("first,starts", [
    (5, [0, 5, -(1 << 31), 0]),                    # the end lies 2^31 and more in front of the beginning
    (5, [0, 5, -(1 << 31) + 4, 0]),
    (5, [0, 5, 3, 3]),                             # and a little in front of it
    (5, [0, 5, (1 << 31) - 1, 0]),                 # ends past the tensor: the tokens that there are
])
@pytest.mark.parametrize("q_lens", [[5, 2, 1], [5, 40, 3]])
def test_offsets_that_go_backwards(q_lens, first, starts, D):
    b = Batch([300, 200, 64], q_lens, 8, 2, D, BF16, seed=30)
    T = b.starts[-1]
    b.qsl = torch.tensor(starts, dtype=torch.int32, device="cuda")
    b.longest_q = max(q_lens)
    b.cross()
    torch.cuda.synchronize()
    assert capi.load_library().device_status() == 0
    live = min(T - first, b.longest_q) if starts[2] > first else 0   # of request 1
    want = reference(b.q, b.k, b.v, b.table, b.kv_lens, [0, first, first + live, first + live], D ** -0.5)
    check(b.out[:first + live], b.lse[:first + live], [w[:first + live] for w in want])
    assert bool(torch.isnan(b.out[first + live:]).all())
    wide = b.out._base if b.out._base is not None else b.out
    assert bool(torch.isnan(wide[:, 0]).all()) and bool(torch.isnan(wide[:, -1]).all())
