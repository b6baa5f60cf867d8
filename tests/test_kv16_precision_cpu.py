"""The bound that the few-row kernel's outputs are held to where they cancel tells P in two 16-bit parts from P in one."""
import pytest
import torch

from tests.kv16_precision import bound, cancel


def _emulate(q, k, v, scale, parts):
    s = torch.einsum("hd,jhd->hj", q.float(), k.float()) * scale
    gain = 2.0 ** (7 if v.dtype == torch.float16 else -24)
    p = torch.exp(s - s.amax(-1, keepdim=True)) * gain
    kept, left = torch.zeros_like(p), p
    for _ in range(parts):
        kept, left = kept + left.to(v.dtype).float(), left - left.to(v.dtype).float()
    return (torch.einsum("hj,jhd->hd", kept, v.float()) / p.sum(-1, keepdim=True)).to(v.dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [3, 40])   # (at 300 keys of 256 dims in fp16 the 32-bit scores' own error hides what one part rounds off)
def test_bound_tells_one_part_from_two(n, D, dtype):
    gen = torch.Generator().manual_seed(n + D)
    q, k, v = ((torch.randn(shape, generator=gen) * x).to(dtype) for shape, x in (((4, D), 0.3), ((n, 4, D), 1.0), ((n, 4, D), 1.0)))
    cancel(q, k, v, D ** -0.5)
    want, tol = bound(q, k, v, D ** -0.5)
    assert bool(((_emulate(q, k, v, D ** -0.5, 2).double() - want).abs() <= tol).all())
    assert bool(((_emulate(q, k, v, D ** -0.5, 1).double() - want).abs() > tol).any())
