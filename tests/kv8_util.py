"""Plain forms of the 8-bit cache's operators, and how far a kernel may be from them."""
from __future__ import annotations

import math

import torch

from tests.kv16_util import ROUNDING, make_table

E4M3 = torch.float8_e4m3fn
LARGEST = 448.0
__all__ = ["E4M3", "LARGEST", "ROUNDING", "make_table", "make_cache", "reference", "check", "write_reference", "read_reference",
           "rotary_reference"]


def make_cache(num_blocks, page, group, Hkv, D, layout="NHD", *, pad=0, device="cuda"):
    """``k_cache``, ``v_cache`` ``[blocks, slots, heads, D]`` and ``k_scale``, ``v_scale`` ``[blocks, slots / group, heads]``: views of
    storages whose pages hold both, with ``pad`` cells behind every row.  All of it is NaN."""
    inner = (page, Hkv) if layout == "NHD" else (Hkv, page)
    cells = torch.full((num_blocks, 2, *inner, D + pad), 0x7f, dtype=torch.uint8, device=device).view(E4M3)
    scales = torch.full((num_blocks, 2, page // group, Hkv + (1 if pad else 0)), math.nan, device=device)
    if layout == "HND":
        cells = cells.transpose(2, 3)
    return cells[:, 0, ..., :D], cells[:, 1, ..., :D], scales[:, 0, :, :Hkv], scales[:, 1, :, :Hkv]


def _gathered(cells, scales, table, at):
    """Cells and scales in 64 bits of positions ``at`` of a request; zero where its block is outside the cache."""
    page, group = cells.shape[1], cells.shape[1] // scales.shape[1]
    blocks = table.long()[at // page]
    known = (blocks >= 0) & (blocks < cells.shape[0])
    b = torch.where(known, blocks, 0)
    c, s = cells[b, at % page].double(), scales[b, at % page // group].double()
    return torch.where(known[:, None, None], c, 0.0), torch.where(known[:, None], s, 0.0)


def _powers_of_two(scale):
    seen = scale[scale.isfinite()]
    return bool((torch.frexp(seen)[0] == 0.5).all())


def reference(q, k_cache, v_cache, k_scale, v_scale, table, kv_lens, starts, scale, window=0, causal=True, tall=False):
    """``out``, ``lse`` in 64 bits, and per element the bound on a kernel's error, from these roundings (e = 2^-24):

    * the result's own, u |out|;
    * queries as sums of e4m3 digits, whose smallest step is 2^-9.  Few rows: digits scaled by 16 each, the row's largest in [128, 256): off
      by 2^-10 / 16 with two (bf16), by 2^-10 / 256 with three (fp16), 2^-21 and 2^-25 of the row's largest.  Many rows (``tall``): digits of one
      unit, the largest in (224, 448]: off by 2^-10, 2^-17 of it.  Times sum |k| in a score;
    * scores: D + 8 32-bit roundings of the sum, and 8 of the score and its distance from the row's bound;
    * weights: fp16, 2^-11 of one.  Few rows: of p scale_V, in digits, off by 2^-18 where they are small, of a row's largest between 2^6 and
      2^8, times the largest scale to the next power of two.  Many rows: of p, off by 2^-25 where they are small, of a largest of 2^7 or
      more; and scale_V c_V in fp16, 2^-11 each of the scale and the product where the scale is no power of two;
    * the sums over n keys, n + 8 roundings, and 2^-21 for the exponentials and the quotient.
    """
    dev = q.device
    T, Hq, D = q.shape
    Hkv, page = k_cache.shape[2], k_cache.shape[1]
    G, u, e = Hq // Hkv, ROUNDING[q.dtype], 2.0 ** -24
    digit = 2.0 ** -17 if tall else 2.0 ** -21 if q.dtype == torch.bfloat16 else 2.0 ** -25
    weight = 2.0 ** -11 + (0.0 if not tall or _powers_of_two(v_scale) else 2.0 ** -10)
    out = torch.zeros((T, Hq, D), dtype=torch.float64, device=dev)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64, device=dev)
    out_tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    for r, seq in enumerate(kv_lens):
        t0, t1 = starts[r], min(starts[r + 1], T)
        n = min(seq, table.shape[1] * page)   # (keys past the row of the table do not exist)
        if t1 <= t0 or n <= 0:
            continue
        at = torch.arange(n, device=dev)
        kc, ks = _gathered(k_cache, k_scale, table[r].to(dev), at)
        vc, vs = _gathered(v_cache, v_scale, table[r].to(dev), at)
        own = torch.arange(seq - (t1 - t0), seq, device=dev)[:, None]
        seen = (at <= own) if causal else torch.ones((t1 - t0, n), dtype=torch.bool, device=dev)
        if window:
            seen = seen & (at > own - window)
        used = seen.any(0)
        k, v = kc * ks[..., None], vc * vs[..., None]
        k, v, vc = (torch.where(used[:, None, None], x, 0.0) for x in (k, v, vc))   # (what nobody sees may be NaN)
        rows = q[t0:t1].double().view(t1 - t0, Hkv, G, D)
        hidden = ~seen[:, None, None]
        s = (torch.einsum("thgd,jhd->thgj", rows, k) * scale).masked_fill(hidden, -math.inf)
        size = (torch.einsum("thgd,jhd->thgj", rows.abs(), k.abs()) * scale).masked_fill(hidden, 0.0)
        far = s.masked_fill(hidden, 0.0).abs().amax(-1)
        digits = digit * rows.abs().amax(-1)[..., None] * (k.abs().sum(-1).t()[:, None] * scale)
        score_err = digits.masked_fill(hidden, 0.0).amax(-1) + (D + 8) * e * size.amax(-1) + 8 * e * 2 * far
        empty = ~seen.any(-1)
        p = torch.softmax(s, -1).masked_fill(empty[:, None, None, None], 0.0)
        o = torch.einsum("thgj,jhd->thgd", p, v)
        spread = torch.einsum("thgj,jhd->thgd", p, v.abs())
        # weights far below the largest: 2^-24 of it (2^-18 / 2^6), times twice the largest scale (the unit is the next power of two)
        small = 2.0 ** -24 * p.amax(-1)[..., None] * 2 * vs.masked_fill(~used[:, None], 0.0).amax(0)[None, :, None, None] \
            * torch.einsum("tj,jhd->thd", seen.double(), vc.abs())[:, :, None]
        sums = (n + 8) * e + 2.0 ** -21
        out[t0:t1] = o.reshape(t1 - t0, Hq, D)
        out_tol[t0:t1] = (u * o.abs() + (weight + 2 * score_err[..., None] + 2 * sums) * spread + small).reshape(t1 - t0, Hq, D)
        logs = torch.logsumexp(s, -1)
        lse[t0:t1] = logs.reshape(t1 - t0, Hq)
        lse_tol[t0:t1] = (score_err + sums + 4 * e * (logs.abs() + 1)).masked_fill(empty[:, None, None], 0.0).reshape(t1 - t0, Hq)
    return out, lse, out_tol, lse_tol


def check(out, lse, want, what=""):
    """Every element within its bound; rows without keys exactly zero, with -inf."""
    ref_out, ref_lse, out_tol, lse_tol = want
    empty = torch.isneginf(ref_lse)
    assert bool((out[empty] == 0).all()), f"{what}: a row without keys is not zero"
    assert bool(torch.isfinite(out).all()), f"{what}: non-finite output"
    tiny = torch.finfo(out.dtype).smallest_normal * ROUNDING[out.dtype] * 2
    d = (out.double() - ref_out).abs()
    over = d - out_tol - tiny
    if over.numel():
        assert float(over.max()) <= 0, f"{what}: out is off by {float(d.flatten()[over.argmax()]):.3e}, bound {float(out_tol.flatten()[over.argmax()]):.3e}"
    if lse.numel():
        assert torch.equal(torch.isneginf(lse), empty), f"{what}: rows without keys differ"
        if not bool(empty.all()):
            dl = ((lse.double() - ref_lse).abs() - lse_tol)[~empty]
            assert float(dl.max()) <= 0, f"{what}: lse is past its bound by {float(dl.max()):.3e}"


def _needed(most):
    """The smallest power of two, 2^-126 to 2^120, with most <= 448 times it."""
    for e in range(-126, 120):
        if most <= LARGEST * 2.0 ** e:
            return 2.0 ** e
    return 2.0 ** 120


def write_reference(key, value, k_cache, v_cache, k_scale, v_scale, table, seq_lens, starts, longest):
    """The caches behind a write, block of tokens by block of tokens (copies on the CPU)."""
    result = [x.cpu().clone() for x in (k_cache, v_cache, k_scale, v_scale)]
    page, group = k_cache.shape[1], k_cache.shape[1] // k_scale.shape[1]
    T = key.shape[0]
    for cells, scales, x in ((result[0], result[2], key.cpu().float()), (result[1], result[3], value.cpu().float())):
        for r, seq in enumerate(seq_lens):
            t0, all_ = starts[r], max(0, min(starts[r + 1], T) - starts[r])
            new = {}   # block of tokens -> [(position, row)]
            for i in range(min(all_, longest)):
                pos = max(0, seq) - all_ + i
                if pos >= 0:
                    new.setdefault(pos // group, []).append((pos, t0 + i))
            for g, tokens in new.items():
                first = tokens[0][0]
                if first // page >= table.shape[1]:
                    continue
                b = int(table[r][first // page])
                if not 0 <= b < cells.shape[0]:
                    continue
                at, n = first % page, first % page // group
                for h in range(cells.shape[2]):
                    rows = torch.stack([x[t, h] for _, t in tokens])
                    finite = rows[rows.isfinite()].abs()
                    need = _needed(float(finite.max()) if finite.numel() else 0.0)
                    was = float(scales[b, n, h])
                    was = was if 0.0 < was < math.inf and at % group else 0.0
                    now = max(was, need)
                    if at % group and now > was:
                        old = cells[b, n * group:at, h].float().double() * was / now
                        cells[b, n * group:at, h] = old.float().to(E4M3)
                    cells[b, at:at + len(tokens), h] = (rows.double() / now).clamp(-LARGEST, LARGEST).float().to(E4M3)
                    scales[b, n, h] = now
    return result


def read_reference(cells, scales, table, first, starts, longest, out):
    """``out`` (a copy) behind a read of one of the two, in 64 bits rounded once."""
    out = out.clone()
    for r, f in enumerate(first):
        rows = min(max(0, starts[r + 1] - starts[r]), longest)
        at = torch.arange(f, f + rows, device=out.device)
        there = (at >= 0) & (at < table.shape[1] * cells.shape[1])
        c, s = _gathered(cells, scales, table[r].to(out.device), torch.where(there, at, 0))
        out[starts[r]:starts[r] + rows] = torch.where(there[:, None, None], c * s[..., None], 0.0).float().to(out.dtype)
    return out


def rotary_reference(x, positions, frequencies, scale, interleaved, inverse):
    """Turned in 64 bits, and the bound on an element's error: its own rounding, and in 32 bits the rounding of the angle (2^-24 pi at
    most, from [-pi, pi]) and of its sine and cosine (2 of their last bits and the scale's), and of two products and a sum."""
    n = frequencies.shape[0]
    angle = torch.outer(positions.double(), frequencies.double()) * (-1.0 if inverse else 1.0)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    out, size = x.double().clone(), x.double().abs()
    a = out[..., 0:2 * n:2] if interleaved else out[..., :n]
    b = out[..., 1:2 * n:2] if interleaved else out[..., n:2 * n]
    a, b = a.clone(), b.clone()
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    out[..., first], out[..., second] = (a * cos - b * sin) * scale, (a * sin + b * cos) * scale
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * abs(scale)
    u = ROUNDING.get(x.dtype, 2.0 ** -24)
    tol = u * out.abs() + (math.pi + 8) * 2.0 ** -24 * size
    if frequencies.dtype == torch.float64 and 2 * n < x.shape[-1]:
        tol[..., 2 * n:] = 0.0
    return out, tol + torch.finfo(x.dtype).smallest_normal * u * 2
