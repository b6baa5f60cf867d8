"""GPU tests of the sines and cosines that rotary positions turn by: as exact near their zeros, where far angles come close to them, as elsewhere."""
import pytest
import torch

from pth_flash_attn_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("base,far", [(10000.0, 0), (1e6, 10 ** 6), (500.0, 10 ** 8)])
def test_unit_vectors(base, far, interleaved):
    """(1, 0) becomes the angle's cosine and sine: 2 of their last bits (the library's sine and cosine of a 32-bit angle), half a bit of the correction, and
    2^-46 of the angle's reduction in 64 bits."""
    gen = torch.Generator().manual_seed(7)
    T, D = 3000, 64
    pos = (torch.randint(0, 100000, (T,), generator=gen) + far).cuda()
    f, _ = ops.rotary_frequencies(D, base, device="cuda")
    q = torch.zeros((T, 1, D), device="cuda")
    first, second = (slice(0, D, 2), slice(1, D, 2)) if interleaved else (slice(0, D // 2), slice(D // 2, D))
    q[..., first] = 1.0
    out, none = torch.empty_like(q), torch.empty((T, 0, D), device="cuda")
    ops.rotary(out, none, q, none, pos, f, 1.0, interleaved)
    angle = torch.outer(pos.double(), f)
    for got, want in ((out[:, 0, first], angle.cos()), (out[:, 0, second], angle.sin())):
        last = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=2.0 ** -126))) - 23)   # distance of neighbouring numbers
        over = (got.double() - want).abs() - 2.5 * last - 2.0 ** -46
        assert float(over.max()) <= 0, f"off by {float(((got.double() - want).abs() / last).max()):.1f} of the last bit"
