"""Plain 64-bit forms of the 16-bit cache's operators, and how far a kernel may be from them."""
from __future__ import annotations

import math

import torch

# largest relative error of one rounding to nearest
ROUNDING = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make_cache(num_blocks, block_size, Hkv, D, dtype, layout="NHD", *, pad=0, gen=None, device="cuda", fill=None):
    """``k_cache`` / ``v_cache`` views ``[blocks, slots, heads, D]`` of one storage whose pages hold both, with ``pad``
    elements behind every row; ``fill`` instead of random values."""
    inner = (block_size, Hkv) if layout == "NHD" else (Hkv, block_size)
    shape = (num_blocks, 2, *inner, D + pad)
    if fill is None:
        storage = torch.randn(shape, generator=gen, device=device).to(dtype)
    else:
        storage = torch.full(shape, fill, dtype=dtype, device=device)
    if layout == "HND":
        storage = storage.transpose(2, 3)
    return storage[:, 0, :, :, :D], storage[:, 1, :, :, :D]


def make_table(kv_lens, block_size, num_blocks, *, gen, width=None):
    """A block table over a shuffled pool; entries that no request needs point outside the cache."""
    pages = [-(-n // block_size) for n in kv_lens]
    assert sum(pages) <= num_blocks
    order = torch.randperm(num_blocks, generator=gen)
    table = torch.full((len(kv_lens), max(1, max(pages, default=1), width or 0)), 1 << 30, dtype=torch.int32)
    first = 0
    for r, n in enumerate(pages):
        table[r, :n] = order[first:first + n].to(torch.int32)
        first += n
    return table


def reference(q, k_cache, v_cache, table, kv_lens, starts, scale, window=0):
    """``out``, ``lse`` in 64 bits, and per element the bound on a kernel's error:

    the result's own rounding u |out|, the rounding of the probabilities to 16 bits, u sum p |v| / sum p, and for both
    contractions 32-bit sums: D + 4 roundings of the scores, whose error moves every p by as much, relatively, and
    n + 8 of the sums over the keys (2^-24 each), with 2^-21 for the exponentials.
    """
    dev = q.device
    T, Hq, D = q.shape
    Hkv, page = k_cache.shape[2], k_cache.shape[1]
    G, u, e = Hq // Hkv, ROUNDING[q.dtype], 2.0 ** -24
    out = torch.zeros((T, Hq, D), dtype=torch.float64, device=dev)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64, device=dev)
    out_tol = torch.zeros_like(out)
    lse_tol = torch.zeros_like(lse)
    for r, n in enumerate(kv_lens):
        t0, t1 = starts[r], min(starts[r + 1], T)
        lo = max(0, n - window) if window else 0
        if t1 <= t0 or n <= lo:
            continue
        at = torch.arange(lo, n, device=dev)
        blocks = table[r].to(dev).long()[at // page]
        k = k_cache[blocks, at % page].double()      # [keys, Hkv, D]
        v = v_cache[blocks, at % page].double()
        rows = q[t0:t1].double().view(t1 - t0, Hkv, G, D)
        s = torch.einsum("thgd,jhd->thgj", rows, k) * scale
        size = torch.einsum("thgd,jhd->thgj", rows.abs(), k.abs()).amax(-1) * scale
        p = torch.softmax(s, -1)
        o = torch.einsum("thgj,jhd->thgd", p, v)
        spread = torch.einsum("thgj,jhd->thgd", p, v.abs())
        score_err = (D + 4) * e * size                       # of one score, absolute (natural units)
        sums = (n - lo + 8) * e + 2.0 ** -21
        out[t0:t1] = o.reshape(t1 - t0, Hq, D)
        out_tol[t0:t1] = (u * o.abs() + (u + 2 * score_err[..., None] + 2 * sums) * spread).reshape(t1 - t0, Hq, D)
        logs = torch.logsumexp(s, -1)
        lse[t0:t1] = logs.reshape(t1 - t0, Hq)
        lse_tol[t0:t1] = (score_err + sums + 4 * e * (logs.abs() + 1)).reshape(t1 - t0, Hq)
    return out, lse, out_tol, lse_tol


def check(out, lse, want, what=""):
    """Every element within its bound; rows without keys exactly zero, with -inf."""
    ref_out, ref_lse, out_tol, lse_tol = want
    empty = torch.isneginf(ref_lse)
    assert torch.equal(torch.isneginf(lse), empty), f"{what}: rows without keys differ"
    assert bool((out[empty] == 0).all()), f"{what}: a row without keys is not zero"
    d = (out.double() - ref_out).abs()
    assert bool(torch.isfinite(out).all()), f"{what}: non-finite output"
    # (a result below the type's smallest normal value rounds to a multiple of its smallest one)
    tiny = torch.finfo(out.dtype).smallest_normal * ROUNDING[out.dtype] * 2
    over = d - out_tol - tiny
    assert float(over.max()) <= 0, f"{what}: out is off by {float(d.flatten()[over.argmax()]):.3e}, bound {float(out_tol.flatten()[over.argmax()]):.3e}"
    if lse.numel() and not bool(empty.all()):
        dl = ((lse.double() - ref_lse).abs() - lse_tol)[~empty]
        assert float(dl.max()) <= 0, f"{what}: lse is past its bound by {float(dl.max()):.3e}"


def tables_reference(context, new, free, table, num_tokens, block_size):
    """The tables of a step, one request, page and token after another."""
    table = [list(map(int, row)) for row in table]
    slots, positions, starts, seq, taken = [-1] * num_tokens, [0] * num_tokens, [0], [], 0
    for r, (c, q) in enumerate(zip(context, new)):
        c, q = max(0, c), max(0, q)
        for page in range(-(-c // block_size), -(-(c + q) // block_size)):
            if page < len(table[r]):
                table[r][page] = free[taken] if taken < len(free) else -1
            taken += 1
        for i in range(q):
            t, pos = starts[-1] + i, c + i
            if t < num_tokens:
                positions[t] = pos
                page = pos // block_size
                if page < len(table[r]) and table[r][page] >= 0:
                    slots[t] = table[r][page] * block_size + pos % block_size
        starts.append(starts[-1] + q)
        seq.append(c + q)
    return table, seq, starts, slots, positions, taken
