"""Batches whose outputs nearly cancel, and how far the few-row kernel may be off there: it keeps probabilities in two 16-bit parts."""
import torch

from tests.kv16_util import ROUNDING


def cancel(q, k, v, scale):
    """Changes the last key's values so that the weighted sum of all is as near to zero as its type allows.  q [Hkv, D], k / v [n, Hkv, D]."""
    p = torch.softmax(torch.einsum("hd,jhd->hj", q.double(), k.double()) * scale, -1)
    rest = torch.einsum("hj,jhd->hd", p[:, :-1], v[:-1].double())
    v[-1] = (-rest / p[:, -1:]).to(v.dtype)


def bound(q, k, v, scale):
    """``out`` of the formula in 64 bits, and per element the bound on the error of a kernel that keeps P in two parts (q [Hkv, D]).

    Of ``kv16_util.reference``'s bound the rounding of P, u sum p |v|, is replaced by that of a remainder, u^2 sum p |v|, and in
    fp16, where P of the largest score is 2^7 at least and the second part is a multiple of 2^-24 (off by 2^-25 at most), by 2^-32 sum |v| more.
    """
    D, n = q.shape[-1], k.shape[0]
    u, e = ROUNDING[v.dtype], 2.0 ** -24
    q, k, dv = q.double(), k.double(), v.double()
    s = torch.einsum("hd,jhd->hj", q, k) * scale
    size = torch.einsum("hd,jhd->hj", q.abs(), k.abs()).amax(-1) * scale
    p = torch.softmax(s, -1)
    o = torch.einsum("hj,jhd->hd", p, dv)
    spread = torch.einsum("hj,jhd->hd", p, dv.abs())
    score_err, sums = (D + 4) * e * size, (n + 8) * e + 2.0 ** -21
    parts = u * u * spread + (2.0 ** -32 * dv.abs().sum(0) if v.dtype == torch.float16 else 0)
    tiny = torch.finfo(v.dtype).smallest_normal * u * 2
    return o, u * o.abs() + parts + (2 * score_err[:, None] + 2 * sums) * spread + tiny
