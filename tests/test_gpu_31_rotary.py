"""GPU tests of rotary positions against their formula in 64 bits, and of the gradient against differences."""
import pytest
import torch

from pth_flash_attn_b200 import ops
from tests.kv8_util import rotary_reference

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _positions(T, far=0):
    gen = torch.Generator().manual_seed(T)
    p = torch.randint(0, 1000, (T,), generator=gen) + far
    return p.cuda()


def _check(got, x, *args):
    want, tol = rotary_reference(x, *args)
    over = (got.double() - want).abs() - tol
    assert float(over.max()) <= 0, f"off by {float((got.double() - want).abs().flatten()[over.argmax()]):.3e}"


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot", [(64, 64), (128, 128), (256, 64), (128, 96), (80, 20), (96, 96), (100, 34), (2, 2), (576, 64), (1024, 1024)])
def test_layouts(D, rot, interleaved, dtype):
    gen = torch.Generator(device="cuda").manual_seed(D)
    T = 37
    q, k = (torch.randn((T, h, D), generator=gen, device="cuda").to(dtype) for h in (5, 2))
    f, _ = ops.rotary_frequencies(rot, device="cuda")
    pos = _positions(T)
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    ops.rotary(q_out, k_out, q, k, pos, f, 1.25, interleaved)
    _check(q_out, q, pos, f, 1.25, interleaved, False)
    _check(k_out, k, pos, f, 1.25, interleaved, False)
    assert torch.equal(q_out[..., rot:], q[..., rot:])


@pytest.mark.parametrize("far", [0, 10 ** 6, 2 ** 31 - 2000, -5000])
@pytest.mark.parametrize("kind", [torch.float64, torch.float32])
def test_far_positions(far, kind):
    gen = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn((20, 4, 128), generator=gen, device="cuda")
    k = torch.randn((20, 1, 128), generator=gen, device="cuda")
    f = ops.rotary_frequencies(128, 1e6, scaling="yarn", factor=8.0, device="cuda")[0].to(kind)
    pos = _positions(20, far)
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    ops.rotary(q_out, k_out, q, k, pos, f)
    _check(q_out, q, pos, f, 1.0, False, False)
    _check(k_out, k, pos, f, 1.0, False, False)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("offset", [0, 1])
def test_strides_in_place_and_parts_of_a_larger_tensor(interleaved, offset):
    """Heads of one projection's output, turned where they are, on 16-byte boundaries and beside them; what lies between stays."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    T, D = 9, 64
    qkv = torch.randn((T, 8 * D + offset), generator=gen, device="cuda").to(BF16)
    before = qkv.clone()

    def parts(x):
        return x[:, offset:offset + 5 * D].unflatten(1, (5, D)), x[:, offset + 5 * D:offset + 6 * D].unflatten(1, (1, D))

    f, _ = ops.rotary_frequencies(D // 2, device="cuda")
    pos = _positions(T)
    q, k = parts(qkv)
    ops.rotary(q, k, q, k, pos, f, 1.0, interleaved)
    for got, x in zip(parts(qkv), parts(before)):
        _check(got, x, pos, f, 1.0, interleaved, False)
    assert torch.equal(qkv[:, offset + 6 * D:], before[:, offset + 6 * D:]) and torch.equal(qkv[:, :offset], before[:, :offset])


def test_inverse_turns_back_and_is_the_gradient():
    gen = torch.Generator(device="cuda").manual_seed(3)
    q, g = (torch.randn((11, 3, 64), generator=gen, device="cuda") for _ in range(2))
    none = torch.empty((11, 0, 64), device="cuda")
    f, _ = ops.rotary_frequencies(48, device="cuda")
    pos = _positions(11, 50000)
    turned, back, grad = torch.empty_like(q), torch.empty_like(q), torch.empty_like(q)
    ops.rotary(turned, none, q, none, pos, f)
    ops.rotary(back, none, turned, none, pos, f, 1.0, False, True)
    assert float((back - q).abs().max()) <= 40 * 2.0 ** -24 * 8   # two turns of up to 20 roundings, of numbers up to 8
    # the gradient of sum(g * turned), scaled: the formula's, and differences of the call itself
    ops.rotary(grad, none, g, none, pos, f, 0.75, False, True)
    _check(grad, g, pos, f, 0.75, False, True)
    x = q.double().requires_grad_()
    n = 24
    angle = torch.outer(pos.double(), f)
    c, s = angle.cos()[:, None] * 0.75, angle.sin()[:, None] * 0.75
    y = torch.cat((x[..., :n] * c - x[..., n:2 * n] * s, x[..., :n] * s + x[..., n:2 * n] * c, x[..., 2 * n:]), -1)
    (y * g.double()).sum().backward()
    assert float((grad.double() - x.grad).abs().max()) <= 20 * 2.0 ** -24 * 8
    step = torch.randn(q.shape, generator=gen, device="cuda")
    plus, minus = torch.empty_like(q), torch.empty_like(q)
    ops.rotary(plus, none, q + step, none, pos, f, 0.75)
    ops.rotary(minus, none, q - step, none, pos, f, 0.75)
    # (turning is linear: differences of any step are exact up to the roundings of numbers up to 8, over 2,112 elements)
    difference = float(((plus.double() - minus.double()) / 2 * g.double()).sum())
    assert abs(difference - float((grad.double() * step.double()).sum())) <= 2112 * 4 * 20 * 2.0 ** -24 * 8


def test_nothing_to_turn():
    f, _ = ops.rotary_frequencies(64, device="cuda")
    e = torch.empty((0, 4, 64), device="cuda")
    ops.rotary(e, e, e, e, torch.empty(0, dtype=torch.int64, device="cuda"), f)
    n = torch.empty((3, 0, 64), device="cuda")
    ops.rotary(n, n, n, n, torch.zeros(3, dtype=torch.int64, device="cuda"), f)
    torch.cuda.synchronize()
