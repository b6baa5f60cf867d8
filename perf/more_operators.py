"""The operators of a block-scaled 8-bit paged cache, as measurable cases with a plain form of each.

Five calls of a serving engine's step, which hand one another their results:

  ``rotary``  ``rotary``: queries and keys turned by their positions;
  ``write``   ``kv8_write``: new tokens' keys and values into a paged e4m3 cache with a scale per block of tokens and head;
  ``read``    ``kv8_read``: a run of cached positions back into 16- or 32-bit rows;
  ``decode``  ``kv8_decode_attention``: one new token of each request over its cache;
  ``attend``  ``kv8_attention``: any number of new tokens of each request over its cache, causal.

A batch is written as text, one term per group of requests: ``count*q+prior``, where ``q`` (tokens of the call;
for ``read`` the positions that are read) and ``prior`` (tokens in front of them) are numbers or ranges ``lo-hi`` drawn
uniformly with ``lens_seed``.  ``8*1+0-4095`` is eight decode requests of 1 to 4,096 keys.
"""
import math
import random

import torch

own = False   # False: elementary torch operations in 32 bits; True: the framework's operators

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_E4M3 = torch.float8_e4m3fn
_LARGEST = 448.0           # e4m3's largest number
_WORKSPACE = 128 << 20     # what an engine keeps for the partial results of split attention calls


def _case(op, batch, Hq=32, Hkv=8, D=128, *, page=64, group=16, layout="NHD", dtype="bf16", window=0, pad=0, lens_seed=1,
          rot=0, interleaved=False, stretch=1.0, name=None):
    """``group``: tokens of a scale; ``rot``: dimensions that turn (0: all); ``stretch``: context that the positions are scaled for."""
    c = dict(op=op, batch=batch, Hq=Hq, Hkv=Hkv, D=D, page=page, group=group, layout=layout, dtype=dtype, window=window, pad=pad,
             lens_seed=lens_seed, rot=rot or D, interleaved=interleaved, stretch=stretch)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # Every step of a decoding batch whose requests are anywhere in a stretched context; half of each head turns.  Latency.
        _case("rotary", "64*1+0-131071", rot=64, interleaved=True, stretch=8.0, name="rotary_decode"),
        # A step that feeds long prompts chunk by chunk, bound by the bytes.
        _case("rotary", "4*2048+30720", name="rotary_chunked"),
        # A decoding step's keys and values: blocks of tokens go on, and some need a larger scale.
        _case("write", "64*1+0-8191", name="write_decode"),
        # A prefill step's keys and values, bound by the bytes.
        _case("write", "4*2048+0", name="write_prefill"),
        # A short prompt's prefix goes to a layer that computes in 16 bits.
        _case("read", "1*1000+0", 12, 2, 256, page=816, group=48, layout="HND", name="read_prefix"),
        # Requests of every length move to another cache.
        _case("read", "16*4096-16384+0-100", dtype="fp16", name="read_requests"),
        # A small interactive batch: launches and the pipeline's fill decide.
        _case("decode", "8*1+0-4095", name="decode_b8"),
        # Throughput serving, bound by the cache's bytes.
        _case("decode", "64*1+8191", name="decode_b64"),
        # Wide heads, few of them, large pages laid out by head; an engine that pads its batch to a captured size.
        _case("decode", "61*1+4095-12287", 12, 2, 256, page=816, group=816, layout="HND", pad=3, name="decode_d256"),
        # Speculative verification: four tokens of every request at a time.
        _case("attend", "32*4+2000-16384", name="verify4"),
        # Prompts of every length with nothing cached, heads of 64.
        _case("attend", "12*37-2500+0", 16, 16, 64, dtype="fp16", page=16, name="prefill_fresh"),
        # Chunks of long prompts over what is cached, bound by the tensor cores.
        _case("attend", "4*2048+8192", name="prefill_chunked"),
    ]


# (query heads, KV heads, head size) met in draws
_HEADS = ((32, 8, 128), (64, 8, 128), (8, 2, 128), (8, 1, 128), (32, 8, 64), (16, 16, 64), (12, 2, 256), (32, 8, 256))
# (slots of a page, tokens of a scale)
_PAGES = ((16, 16), (32, 16), (48, 48), (64, 16), (64, 64), (128, 32), (816, 48), (816, 816))


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def _span(rng, hi, lo=0):
    """All requests alike, or ragged from ``lo`` (or anything between) up to ``hi``."""
    if rng.random() < 0.25:
        return str(hi)
    low = lo + round((hi - lo) * rng.choice((0.0, rng.random())))
    return f"{low}-{hi}" if low < hi else str(hi)


def _draw_any(rng):
    op = rng.choice(("rotary", "write", "read", "decode", "decode", "attend", "attend"))
    Hq, Hkv, D = rng.choice(_HEADS)
    page, group = rng.choice(_PAGES)
    opt = dict(page=page, group=group, layout=rng.choice(("NHD", "HND")), dtype=rng.choice(("bf16", "bf16", "fp16")),
               lens_seed=rng.randrange(1 << 30), pad=rng.choice((0, 0, rng.randint(1, 5))))
    few = rng.random() < 0.4
    if op in ("rotary", "write"):
        if few:
            batch = f"{_log_int(rng, 1, 512)}*1+{_span(rng, _log_int(rng, 16, 131072))}"
        else:
            batch = f"{_log_int(rng, 1, 64)}*{_span(rng, _log_int(rng, 16, 4096), 1)}+{_span(rng, _log_int(rng, 16, 16384))}"
        opt["dtype"] = rng.choice((opt["dtype"], opt["dtype"], "fp32"))
        if op == "rotary":
            opt |= dict(rot=rng.choice((D, D, D // 2, D // 4)), interleaved=rng.random() < 0.5, stretch=rng.choice((1.0, 1.0, 4.0, 16.0)))
        return _case(op, batch, Hq, Hkv, D, **opt)
    if op == "read":
        opt["dtype"] = rng.choice((opt["dtype"], opt["dtype"], "fp32"))
        batch = f"{_log_int(rng, 1, 64)}*{_span(rng, _log_int(rng, 16, 16384), 1)}+{_span(rng, _log_int(rng, 1, 4096))}"
        return _case(op, batch, Hq, Hkv, D, **opt)
    opt["window"] = rng.choice((0, 0, 0, rng.randint(128, 4096)))
    if op == "decode":
        return _case(op, f"{_log_int(rng, 1, 256)}*1+{_span(rng, _log_int(rng, 16, 131071))}", Hq, Hkv, D, **opt)
    q = _span(rng, _log_int(rng, 2, 16 if few else 2048), 1)
    return _case(op, f"{_log_int(rng, 1, 64)}*{q}+{_span(rng, _log_int(rng, 16, 16384))}", Hq, Hkv, D, **opt)


def draw(rng):
    """A case of the listed cases' ranges, no heavier in bytes or in operations than the heaviest of them."""
    heaviest = [max(work(c)[unit] for c in listed()) for unit in ("bytes", "flops")]
    while True:
        case = _draw_any(rng)
        w = work(case)
        lengths = _lengths(case)
        longest_q, longest = max(q for q, _ in lengths), max(n for _, n in lengths)
        # (the plain form of attention pads every request to the longest)
        padded = len(lengths) * longest * max(case["Hkv"] * case["D"] * 4, case["Hq"] * longest_q) if case["op"] in ("decode", "attend") else 0
        pool = sum(n for _, n in lengths) * case["Hkv"] * case["D"] if case["op"] not in ("rotary", "write") else 0
        if w["bytes"] <= heaviest[0] and w["flops"] <= heaviest[1] and padded <= 1 << 32 and pool <= 1 << 31:
            return case


def _range(text, rng):
    lo, _, hi = text.partition("-")
    return rng.randint(int(lo), int(hi)) if hi else int(lo)


def _lengths(case):
    """(tokens of the call, tokens with them) of every request; ``pad`` requests without either fill up the batch."""
    rng = random.Random(case["lens_seed"])
    out = []
    for term in case["batch"].split():
        count, _, rest = term.partition("*")
        q, _, prior = rest.partition("+")
        for _ in range(int(count)):
            n, before = _range(q, rng), _range(prior, rng)
            out.append((n, before + n))
    return out + [(0 if case["op"] != "decode" else 1, 0)] * case["pad"]


def _size(case):
    return 4 if case["dtype"] == "fp32" else 2


def _seen(q, n, window):
    """Cells that the last q of n tokens see together, and (token, key) pairs."""
    if not window:
        return n, q * (n - q) + q * (q + 1) // 2
    return min(n, window + q - 1), sum(min(window, n - i) for i in range(q))


def work(case):
    """Queries, outputs and every visible cell with its scales once; two contractions per visible (query, key) pair."""
    D, Hq, Hkv, page, group = case["D"], case["Hq"], case["Hkv"], case["page"], case["group"]
    lengths = _lengths(case)
    R, tokens = len(lengths), sum(q for q, _ in lengths)
    if case["op"] == "rotary":
        return {"bytes": 2 * tokens * (Hq + Hkv) * D * _size(case) + 8 * tokens, "flops": 3 * tokens * (Hq + Hkv) * case["rot"]}
    if case["op"] == "write":   # a block of tokens that goes on is read too
        old = sum((n - q) % group for q, n in lengths if q)
        blocks = sum(-(-n // group) - (n - q) // group for q, n in lengths if q)
        return {"bytes": 2 * Hkv * (tokens * D * (_size(case) + 1) + old * D + 4 * blocks) + 8 * R, "flops": 4 * tokens * Hkv * D}
    if case["op"] == "read":
        blocks = sum(-(-n // group) - (n - q) // group for q, n in lengths if q)
        return {"bytes": 2 * Hkv * (tokens * D * (_size(case) + 1) + 4 * blocks) + 12 * R, "flops": 2 * tokens * Hkv * D}
    seen = [_seen(q, n, case["window"]) for q, n in lengths if q and n]
    cells = sum(c for c, _ in seen)
    return {"bytes": cells * 2 * Hkv * D + 8 * Hkv * -(-cells // group) + 4 * -(-cells // page) + 4 * tokens * Hq * D + 4 * tokens * Hq + 8 * R,
            "flops": 4 * D * Hq * sum(p for _, p in seen)}


def _int32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _starts(lengths, device):
    return torch.tensor([0] + [q for q, _ in lengths], device=device).cumsum(0).to(torch.int32)


def _pages(case, first, lengths, gen, device):
    """A shuffled pool of pages: the table of what each request needs from position first[r] on, and the pool's size."""
    page = case["page"]
    lo = torch.tensor([f // page for f in first], device=device)
    hi = torch.tensor([-(-n // page) for _, n in lengths], device=device)
    at = torch.arange(max(1, int(hi.max())), device=device)
    needed = (at >= lo[:, None]) & (at < hi[:, None])
    total = int(needed.sum())
    table = torch.zeros(needed.shape, dtype=torch.int32, device=device)
    table[needed] = torch.randperm(total, generator=gen, device=device).to(torch.int32)
    return table, max(1, total)


def _cache(case, blocks, gen, device):
    """Cells and scales of a layer's keys or values: views [blocks, slots, heads, D] and [blocks, slots / group, heads]."""
    D, Hkv, page = case["D"], case["Hkv"], case["page"]
    shape = (blocks, page, Hkv, D) if case["layout"] == "NHD" else (blocks, Hkv, page, D)
    cells = torch.empty(shape, dtype=_E4M3, device=device)
    per = max(1, (1 << 26) // (page * Hkv * D))
    for b in range(0, blocks, per):   # (piece by piece: a whole pool in 32 bits would take four times its room)
        part = cells[b:b + per]
        part.copy_(torch.randn(part.shape, generator=gen, device=device).mul_(100.0).clamp_(-_LARGEST, _LARGEST))
    if case["layout"] == "HND":
        cells = cells.transpose(1, 2)
    # powers of two around what unit normal values need
    exponent = torch.randint(-8, -5, (blocks, page // case["group"], Hkv), generator=gen, device=device)
    return cells, torch.exp2(exponent.float())


def _frequencies(case, device):
    """Radians per position: slow dimensions are stretched, fast ones kept, those between blended."""
    rot, stretch, trained = case["rot"], case["stretch"], 4096
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    turns = trained * f / (2 * math.pi)
    keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
    return f * keep + f / stretch * (1.0 - keep), 0.1 * math.log(stretch) + 1.0


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    lengths = _lengths(case)
    R, T, D, Hq, Hkv, page = len(lengths), sum(q for q, _ in lengths), case["D"], case["Hq"], case["Hkv"], case["page"]
    kind, op = _DTYPES[case["dtype"]], case["op"]
    starts, longest_q = _starts(lengths, device), max(q for q, _ in lengths)

    def rows(heads):
        return torch.randn((T, heads, D), generator=gen, device=device).to(kind)

    if op == "rotary":
        positions = torch.cat([torch.arange(n - q, n, device=device) for q, n in lengths])
        q, k = rows(Hq), rows(Hkv)
        f, scale = _frequencies(case, device)
        return dict(op=op, q=q, k=k, q_out=torch.empty_like(q), k_out=torch.empty_like(k), positions=positions, frequencies=f,
                    scale=scale, interleaved=case["interleaved"])

    needed = [0 if op in ("decode", "attend") else n - q for q, n in lengths]
    table, blocks = _pages(case, needed, lengths, gen, device)
    (k_cache, k_scale), (v_cache, v_scale) = (_cache(case, blocks, gen, device) for _ in range(2))
    state = dict(op=op, k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, block_table=table,
                 seq_lens=_int32([n for _, n in lengths], device), query_start_loc=starts, longest_q=longest_q)
    if op == "write":
        # channels of keys differ in size, and so do tokens
        spread = torch.exp(torch.randn((1, Hkv, D), generator=gen, device=device) * 0.7)
        size = torch.exp(torch.randn((T, 1, 1), generator=gen, device=device) * 0.5)
        return state | dict(key=(rows(Hkv) * spread * size).to(kind), value=(rows(Hkv) * size).to(kind))
    if op == "read":
        return state | dict(first=_int32([n - q for q, n in lengths], device),
                            key=torch.zeros((T, Hkv, D), dtype=kind, device=device), value=torch.zeros((T, Hkv, D), dtype=kind, device=device))
    q = rows(Hq)
    return state | dict(q=q, scale=D ** -0.5, window=case["window"], longest=max(n for _, n in lengths), out=torch.zeros_like(q),
                        lse=torch.zeros((T, Hq), dtype=torch.float32, device=device),
                        workspace=torch.zeros(_WORKSPACE, dtype=torch.uint8, device=device))


def run(state):
    return _RUN[state["op"]](state)


def _run_rotary(s):
    if own:
        from pth_flash_attn_b200 import ops
        ops.rotary(s["q_out"], s["k_out"], s["q"], s["k"], s["positions"], s["frequencies"], s["scale"], s["interleaved"])
        return {"q": s["q_out"], "k": s["k_out"]}
    angle = s["positions"].double()[:, None] * s["frequencies"]
    cos, sin = ((t * s["scale"]).float()[:, None] for t in (angle.cos(), angle.sin()))
    half = cos.shape[-1]
    out = {}
    for name in ("q", "k"):
        x = s[name].float()
        turning, rest = x[..., :2 * half], x[..., 2 * half:]
        a, b = (turning[..., ::2], turning[..., 1::2]) if s["interleaved"] else (turning[..., :half], turning[..., half:])
        a, b = a * cos - b * sin, a * sin + b * cos
        turned = torch.stack((a, b), -1).flatten(-2) if s["interleaved"] else torch.cat((a, b), -1)
        out[name] = torch.cat((turned, rest), -1).to(s[name].dtype)
    return out


def _places(s, first, starts, rows):
    """Block and slot of `rows` rows: row starts[r] + i is position first[r] + i of request r."""
    page, starts = s["k_cache"].shape[1], starts.long()
    req = torch.searchsorted(starts[1:], torch.arange(rows, device=starts.device), right=True)
    at = torch.arange(rows, device=starts.device) - starts[req] + first.long()[req]
    return s["block_table"][req, at // page].long(), at % page


def _run_write(s):
    if own:
        from pth_flash_attn_b200 import ops
        ops.kv8_write(s["key"], s["value"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["block_table"], s["seq_lens"],
                      s["query_start_loc"], s["longest_q"])
        return {n: s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
    starts = s["query_start_loc"]
    block, slot = _places(s, s["seq_lens"] - (starts[1:] - starts[:-1]), starts, len(s["key"]))
    page, groups = s["k_cache"].shape[1], s["k_scale"].shape[1]
    g = page // groups
    # the blocks of tokens that are written to, and the first slot of them that is
    ids, which = (block * groups + slot // g).unique(return_inverse=True)
    first = torch.full_like(ids, g).scatter_reduce(0, which, slot % g, "amin")
    b, n = ids // groups, ids % groups
    within = torch.arange(g, device=ids.device)
    older = within < first[:, None]
    for cells, scales, x in ((s["k_cache"], s["k_scale"], s["key"].float()), (s["v_cache"], s["v_scale"], s["value"].float())):
        size = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
        most = torch.zeros((len(ids), size.shape[1]), device=x.device).scatter_reduce(0, which[:, None].expand_as(size), size, "amax")
        mantissa, exponent = torch.frexp(most / _LARGEST)   # a scale is the power of two at or above it
        needed = torch.exp2((exponent - (mantissa == 0.5).int()).clamp(-126, 120).float())
        needed = torch.where(most > 0, needed, 2.0 ** -126)
        was = scales[b, n]
        now = torch.where(first[:, None] == 0, needed, torch.maximum(was, needed))
        where = (b[:, None].expand_as(older)[older], (n[:, None] * g + within)[older])
        ratio = (was / now)[:, None].expand(-1, g, -1)[older]
        cells[where] = (cells[where].float() * ratio[..., None]).to(_E4M3)
        cells[block, slot] = (x / now[which][..., None]).clamp(-_LARGEST, _LARGEST).to(_E4M3)
        scales[b, n] = now
    return {n: s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}


def _run_read(s):
    if own:
        from pth_flash_attn_b200 import ops
        ops.kv8_read(s["key"], s["value"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["block_table"], s["first"],
                     s["query_start_loc"], s["longest_q"])
        return {"key": s["key"], "value": s["value"]}
    block, slot = _places(s, s["first"], s["query_start_loc"], len(s["key"]))
    group = slot // (s["k_cache"].shape[1] // s["k_scale"].shape[1])
    return {"key": (s["k_cache"][block, slot].float() * s["k_scale"][block, group][..., None]).to(s["key"].dtype),
            "value": (s["v_cache"][block, slot].float() * s["v_scale"][block, group][..., None]).to(s["value"].dtype)}


def _run_decode(s):
    if own:
        from pth_flash_attn_b200 import ops
        ops.kv8_decode_attention(s["out"], s["lse"], s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["block_table"],
                                 s["seq_lens"], s["scale"], s["workspace"], s["window"])
        return {"out": s["out"], "lse": s["lse"]}
    q, (R, Hq, D) = s["q"], s["q"].shape
    keys, values, at = _gather(s)
    seen = at < s["seq_lens"][:, None]
    if s["window"]:
        seen &= at >= (s["seq_lens"] - s["window"])[:, None]
    out, lse = _attend(q.float().view(R, -1, Hq // keys.shape[1], D), keys, values, seen[:, None, None], s["scale"])
    return {"out": out.reshape(R, Hq, D).to(q.dtype), "lse": lse.reshape(R, Hq)}


def _run_attend(s):
    if own:
        from pth_flash_attn_b200 import ops
        ops.kv8_attention(s["out"], s["lse"], s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["block_table"], s["seq_lens"],
                          s["query_start_loc"], s["longest_q"], s["scale"], s["workspace"], s["window"])
        return {"out": s["out"], "lse": s["lse"]}
    q, (T, Hq, D) = s["q"], s["q"].shape
    keys, values, at = _gather(s)
    R, Hkv = keys.shape[:2]
    starts, G, n = s["query_start_loc"].long(), Hq // keys.shape[1], s["longest_q"]
    i = torch.arange(n, device=q.device)
    q_lens = starts[1:] - starts[:-1]
    token, live = starts[:-1, None] + i, i < q_lens[:, None]
    last = (s["seq_lens"] - q_lens)[:, None] + i   # the last key that token i sees
    seen = (at <= last[..., None]) & (at < s["seq_lens"][:, None, None])
    if s["window"]:
        seen &= at > last[..., None] - s["window"]
    rows = q[token.clamp(max=T - 1)].float().view(R, n, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(R, Hkv, G * n, D)
    seen = seen[:, None, None].expand(-1, 1, G, -1, -1).reshape(R, 1, G * n, -1)
    out, lse = _attend(rows, keys, values, seen, s["scale"])
    out = out.view(R, Hkv, G, n, D).permute(0, 3, 1, 2, 4).reshape(R, n, Hq, D)
    lse = lse.view(R, Hkv, G, n).permute(0, 3, 1, 2).reshape(R, n, Hq)
    return {"out": out[live].to(q.dtype), "lse": lse[live]}


def _gather(s):
    """Keys and values [R, Hkv, keys, D] of every request up to the longest, and the positions."""
    page, table = s["k_cache"].shape[1], s["block_table"]
    at = torch.arange(s["longest"], device=table.device)
    block, slot = table[:, at // page].long(), at % page
    group = slot // (page // s["k_scale"].shape[1])
    keys = s["k_cache"][block, slot].float().mul_(s["k_scale"][block, group][..., None])
    values = s["v_cache"][block, slot].float().mul_(s["v_scale"][block, group][..., None])
    return keys.transpose(1, 2), values.transpose(1, 2), at


def _attend(rows, keys, values, seen, scale):
    """rows [R, Hkv, rows, D] over keys: the output and the log-sum-exp; a row that sees no key is 0 and -inf."""
    scores = (rows @ keys.transpose(2, 3)).mul_(scale).masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p @ values) / total.clamp(min=torch.finfo(torch.float32).tiny)
    return out, torch.where(total > 0, top + total.log(), -math.inf)[..., 0]


_RUN = {"rotary": _run_rotary, "write": _run_write, "read": _run_read, "decode": _run_decode, "attend": _run_attend}


def exact(case, seed):
    """The same in 64 bits, request by request and block by block."""
    if case["op"] == "write" and sum(q for q, _ in _lengths(case)) > 40000:
        return None
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "write": _exact_write, "read": _exact_read, "decode": _exact_attention, "attend": _exact_attention}[case["op"]](case, s)


def _exact_rotary(case, s):
    rot = case["rot"]
    angle = torch.outer(s["positions"].double(), s["frequencies"])
    turn = torch.complex(angle.cos(), angle.sin())[:, None] * s["scale"]
    first = torch.arange(0, rot, 2, device="cuda") if case["interleaved"] else torch.arange(rot // 2, device="cuda")
    second = first + 1 if case["interleaved"] else first + rot // 2
    out = {}
    for name in ("q", "k"):
        x = s[name].double()
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        out[name] = x
    return out


def _exact_write(case, s):
    """Scales by comparison with every power of two; values as quotients, not rounded."""
    g, page = case["group"], case["page"]
    powers = torch.exp2(torch.arange(-126, 121, device="cuda").double())
    result = {n: s[n].double() for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
    starts = s["query_start_loc"].tolist()
    blocks = []   # (first position of the request's tokens in the block of tokens, their number, first row, block, group)
    table = s["block_table"].cpu()
    for r, (q, n) in enumerate(_lengths(case)):
        at = n - q
        while at < n:
            count = min(n, (at // g + 1) * g) - at
            blocks.append((at % g, count, starts[r] + at - (n - q), int(table[r, at // page]), at % page // g))
            at += count
    for cells, scales, x in (("k_cache", "k_scale", s["key"]), ("v_cache", "v_scale", s["value"])):
        c, sc, x = result[cells], result[scales], x.double()
        for begin, count, row, b, n in blocks:
            new = x[row:row + count]
            scale = powers[torch.searchsorted(powers, new.abs().amax((0, 2)) / 448.0).clamp(max=246)]
            at = n * g + begin
            if begin:
                old = sc[b, n].clone()
                scale = torch.maximum(scale, old)
                c[b, n * g:at] *= (old / scale)[:, None]
            c[b, at:at + count] = new / scale[:, None]
            sc[b, n] = scale
    return result


def _exact_read(case, s):
    out = {n: torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in ("key", "value")}
    row = 0
    for r, (q, n) in enumerate(_lengths(case)):
        at = torch.arange(n - q, n, device="cuda")
        b, slot = s["block_table"][r].long()[at // case["page"]], at % case["page"]
        for name, cells, scales in (("key", "k_cache", "k_scale"), ("value", "v_cache", "v_scale")):
            out[name][row:row + q] = s[cells][b, slot].double() * s[scales].double()[b, slot // case["group"]][..., None]
        row += q
    return out


def _exact_attention(case, s):
    G, D, page, group, window = case["Hq"] // case["Hkv"], case["D"], case["page"], case["group"], case["window"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    begin = 0
    for r, (q, n) in enumerate(_lengths(case)):
        tokens = slice(begin, begin + q)
        begin += q
        if n == 0 or q == 0:
            continue
        low = max(0, n - q + 1 - window) if window else 0
        at = torch.arange(low, n, device="cuda")
        b, slot = s["block_table"][r].long()[at // page], at % page
        own_position = torch.arange(n - q, n, device="cuda")[:, None]
        hidden = at > own_position
        if window:
            hidden |= at <= own_position - window
        for h in range(case["Hkv"]):
            heads = slice(h * G, (h + 1) * G)
            k, v = (s[cells][:, :, h][b, slot].double() * s[scales][:, :, h][b, slot // group].double()[:, None]
                    for cells, scales in (("k_cache", "k_scale"), ("v_cache", "v_scale")))
            scores = torch.einsum("thd,jd->thj", s["q"][tokens, heads].double(), k) / math.sqrt(D)
            scores.masked_fill_(hidden[:, None], -math.inf)
            lse[tokens, heads] = torch.logsumexp(scores, -1)
            out[tokens, heads] = torch.einsum("thj,jd->thd", torch.softmax(scores, -1), v)
    return {"out": out, "lse": lse}
