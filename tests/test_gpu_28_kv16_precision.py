"""GPU test that the few-row kernel of the 16-bit cache keeps probabilities in two 16-bit parts: where an output's terms cancel, what one part
rounds off is more than the bound allows (``test_kv16_precision_cpu.py`` holds the bound to that)."""
import pytest
import torch

from tests.kv16_precision import bound, cancel
from tests.test_gpu_20_kv16_attention import BF16, F16, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("G", [1, 4, 8, 16, 32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("form", ["decode", "cross"])
def test_outputs_that_cancel(form, D, G, dtype):
    kv_lens = [3, 40, 300, 5000]
    b = Batch(kv_lens, [1] * 4, 2 * G, 2, D, dtype, scale_up=0.3, seed=D + G)
    b.q.copy_(b.q[:, ::G].repeat_interleave(G, 1))   # (all rows of a KV head alike: they cancel together)
    wants = []
    for r, n in enumerate(kv_lens):
        at = torch.arange(n)
        where = b.table[r].long()[at // b.page].cuda(), (at % b.page).cuda()
        k, v, q = b.k[where], b.v[where], b.q[r, ::G]
        cancel(q, k, v, D ** -0.5)
        b.v[where] = v
        wants.append(bound(q, k, v, D ** -0.5))
    b.decode() if form == "decode" else b.cross()
    torch.cuda.synchronize()
    for r, (want, tol) in enumerate(wants):
        off = (b.out[r].double() - want.repeat_interleave(G, 0)).abs() / tol.repeat_interleave(G, 0)
        assert float(off.max()) <= 1, f"{kv_lens[r]} keys: {float(off.max()):.2f} of the bound"
