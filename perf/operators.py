"""The operators of a 16-bit paged cache, as measurable cases with a plain form of each.

Four calls of a serving engine's step, which hand one another their results:

  ``tables``  ``page_tables``: block table, slot map, positions and start offsets from the requests' lengths;
  ``write``   ``kv16_write``: the keys and values of new tokens into a paged cache of 16-bit cells;
  ``decode``  ``kv16_decode_attention``: one new token of each request over its cache;
  ``cross``   ``kv16_cross_attention``: a request's query tokens over the states of its encoder, which lie in pages too.

A batch is written as text, one term per group of requests: ``count*q+prior``, where ``q`` (query tokens of
the call) and ``prior`` (tokens already in the cache; for ``cross`` the encoder's states) are numbers or ranges
``lo-hi`` drawn uniformly with ``lens_seed``.  ``8*1+0-4095`` is eight decode requests of 1 to 4,096 keys.
"""
import math
import random

import torch

own = False   # False: elementary torch operations in 32 bits; True: the framework's operators

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_WORKSPACE = 64 << 20   # what an engine keeps for the partial results of split attention calls


def _case(op, batch, Hq=32, Hkv=8, D=128, *, page=16, layout="NHD", dtype="bf16", src=None, window=0, pad=0, lens_seed=1,
          name=None):
    c = dict(op=op, batch=batch, Hq=Hq, Hkv=Hkv, D=D, page=page, layout=layout, dtype=dtype, src=src or dtype, window=window,
             pad=pad, lens_seed=lens_seed)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # Every step of a decoding batch: one token per request, seldom a new page.  Latency alone.
        _case("tables", "64*1+8191", name="tables_decode"),
        # A step that feeds long prompts chunk by chunk.
        _case("tables", "4*2048+30720", name="tables_chunked"),
        # A batch of documents of every length is admitted at once.
        _case("tables", "128*37-2500+0", name="tables_admit"),
        # The same decoding step's keys and values: little data, latency.
        _case("write", "64*1+8191", name="write_decode"),
        # A prefill step's keys and values, bound by the bytes.
        _case("write", "4*2048+0", name="write_prefill"),
        # A small interactive batch: launches and the pipeline's fill decide.
        _case("decode", "8*1+0-4095", name="decode_b8"),
        # One very long document being continued: all the parallelism has to come from the keys.
        _case("decode", "1*1+131071", name="decode_long_b1"),
        # Throughput serving, bound by the cache's bytes.
        _case("decode", "64*1+8191", name="decode_b64"),
        # Wide heads, few of them, large pages that are laid out by head; an engine that pads its batch to a captured size.
        _case("decode", "61*1+4095-12287", 12, 2, 256, page=816, layout="HND", pad=3, name="decode_d256"),
        # A decoder's layer that looks at its encoder, token by token: every request has states of its own length.
        _case("cross", "64*1+64-1500", 16, 16, 64, dtype="fp16", name="cross_token"),
        # Prompts of such decoders: ragged on both sides.
        _case("cross", "16*4-448+64-1500", 16, 16, 64, name="cross_prompt"),
        # Long queries over long documents, bound by the tensor cores.
        _case("cross", "4*2048+8192", name="cross_long"),
    ]


# (query heads, KV heads, head size) met in draws
_HEADS = ((32, 8, 128), (64, 8, 128), (8, 2, 128), (8, 1, 128), (32, 8, 64), (16, 16, 64), (12, 2, 256), (32, 8, 256))


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def _span(rng, hi, lo=0):
    """All requests alike, or ragged from ``lo`` (or anything between) up to ``hi``."""
    if rng.random() < 0.25:
        return str(hi)
    low = lo + round((hi - lo) * rng.choice((0.0, rng.random())))
    return f"{low}-{hi}" if low < hi else str(hi)


def _draw_any(rng):
    op = rng.choice(("tables", "write", "decode", "decode", "cross", "cross"))
    Hq, Hkv, D = rng.choice(_HEADS)
    opt = dict(layout=rng.choice(("NHD", "HND")), dtype=rng.choice(("bf16", "bf16", "fp16")),
               page=rng.choice((16, 16, 24, 32, 64, 816)), lens_seed=rng.randrange(1 << 30), pad=rng.choice((0, 0, rng.randint(1, 5))))
    if op in ("tables", "write"):
        if rng.random() < 0.4:
            batch = f"{_log_int(rng, 1, 512)}*1+{_span(rng, _log_int(rng, 16, 16384))}"
        else:
            batch = f"{_log_int(rng, 1, 64)}*{_span(rng, _log_int(rng, 16, 4096), 1)}+{_span(rng, _log_int(rng, 16, 16384))}"
        src = rng.choice((opt["dtype"], opt["dtype"], "fp32"))
        return _case(op, batch, Hq, Hkv, D, **opt, src=src)
    if op == "decode":
        batch = f"{_log_int(rng, 1, 256)}*1+{_span(rng, _log_int(rng, 16, 131071))}"
        return _case(op, batch, Hq, Hkv, D, **opt, window=rng.choice((0, 0, 0, rng.randint(128, 4096))))
    q = rng.choice(("1", _span(rng, _log_int(rng, 2, 2048), 1)))
    batch = f"{_log_int(rng, 1, 64)}*{q}+{_span(rng, _log_int(rng, 16, 16384))}"
    return _case(op, batch, Hq, Hkv, D, **opt)


def draw(rng):
    """A case of the listed cases' ranges, no heavier in bytes or in operations than the heaviest of them."""
    heaviest = [max(work(c)[unit] for c in listed()) for unit in ("bytes", "flops")]
    while True:
        case = _draw_any(rng)
        w = work(case)
        lengths = _lengths(case)
        longest_q, longest = max(q for q, _ in lengths), max(n for _, n in lengths)
        # (the plain form pads every request to the longest)
        padded = len(lengths) * longest * (case["Hkv"] * case["D"] * 4 if case["op"] != "cross" else case["Hq"] * longest_q)
        pool = sum(n for _, n in lengths) * case["Hkv"] * case["D"]
        if w["bytes"] <= heaviest[0] and w["flops"] <= heaviest[1] and padded <= 1 << 32 and pool <= 1 << 31:
            return case


def _range(text, rng):
    lo, _, hi = text.partition("-")
    return rng.randint(int(lo), int(hi)) if hi else int(lo)


def _lengths(case):
    """(query tokens, keys) of every request of the call; ``pad`` requests without either fill up the batch."""
    rng = random.Random(case["lens_seed"])
    out = []
    for term in case["batch"].split():
        count, _, rest = term.partition("*")
        q, _, prior = rest.partition("+")
        for _ in range(int(count)):
            n, before = _range(q, rng), _range(prior, rng)
            out.append((n, before if case["op"] == "cross" else before + n))
    return out + [(0 if case["op"] != "decode" else 1, 0)] * case["pad"]


def work(case):
    """Lengths, tables, queries, outputs and every visible cell once; two contractions per visible (query, key) pair."""
    D, Hq, Hkv, page, window = case["D"], case["Hq"], case["Hkv"], case["page"], case["window"]
    lengths = _lengths(case)
    R, tokens = len(lengths), sum(q for q, _ in lengths)
    if case["op"] == "tables":   # two lengths and the page that goes on in; two offsets out; new pages in and out; slots and positions out
        pages = sum(-(-n // page) - -(-(n - q) // page) for q, n in lengths)
        return {"bytes": 20 * R + 8 * pages + 16 * tokens, "flops": 8 * tokens + 8 * R}
    if case["op"] == "write":
        source = 4 if case["src"] == "fp32" else 2
        return {"bytes": tokens * (2 * Hkv * D * (source + 2) + 8), "flops": 2 * tokens * Hkv * D}
    seen = [min(n, window) if window else n for _, n in lengths]
    cells = sum(n for (q, _), n in zip(lengths, seen) if q)
    pairs = sum(q * n for (q, _), n in zip(lengths, seen))
    return {"bytes": cells * 4 * Hkv * D + 4 * -(-cells // page) + 4 * tokens * Hq * D + 4 * tokens * Hq + 8 * R,
            "flops": 4 * D * Hq * pairs}


def _pages(case, lengths, gen, device, spare=0):
    """A shuffled pool of pages: the table of what each request holds (all of its keys), and the ids that are left."""
    page = case["page"]
    held = torch.tensor([-(-n // page) for _, n in lengths], device=device)
    total = int(held.sum())
    order = torch.randperm(total + spare, generator=gen, device=device).to(torch.int32)
    width = max(1, int(held.max()))
    table = torch.zeros((len(lengths), width), dtype=torch.int32, device=device)
    table[torch.arange(width, device=device) < held[:, None]] = order[:total]
    return table, order[total:], total + spare


def _caches(case, blocks, gen, device):
    """Keys and values of a layer as views [blocks, slots, heads, D] of one storage, in one of the two page layouts."""
    D, Hkv, page = case["D"], case["Hkv"], case["page"]
    inner = (page, Hkv) if case["layout"] == "NHD" else (Hkv, page)
    storage = torch.randn((2, blocks, *inner, D), generator=gen, device=device, dtype=_DTYPES[case["dtype"]])
    if case["layout"] == "HND":
        storage = storage.transpose(2, 3)
    return storage[0], storage[1]


def _int32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    lengths = _lengths(case)
    R, T, D, Hq, Hkv, page = len(lengths), sum(q for q, _ in lengths), case["D"], case["Hq"], case["Hkv"], case["page"]
    q_lens, kv_lens = [q for q, _ in lengths], [n for _, n in lengths]

    if case["op"] == "tables":
        # what the requests hold before the step; the new pages come off a list of free ones
        before = [(q, n - q) for q, n in lengths]
        new = sum(-(-n // page) for n in kv_lens) - sum(-(-n // page) for _, n in before)
        held, free, _ = _pages(case, before, gen, device, spare=new + 64)
        table = torch.zeros((R, -(-max(kv_lens) // page) + 1), dtype=torch.int32, device=device)
        table[:, :held.shape[1]] = held
        padded = T + case["pad"]   # a captured step's token arrays are as long as its largest batch
        return dict(op="tables", page=page, context_lens=_int32([n for _, n in before], device), query_lens=_int32(q_lens, device),
                    free_blocks=free, block_table=table, seq_lens=torch.zeros(R, dtype=torch.int32, device=device),
                    query_start_loc=torch.zeros(R + 1, dtype=torch.int32, device=device),
                    slot_mapping=torch.zeros(padded, dtype=torch.int64, device=device),
                    positions=torch.zeros(padded, dtype=torch.int64, device=device),
                    pages_taken=torch.zeros(1, dtype=torch.int32, device=device))

    if case["op"] == "write":
        # the step's slots: the last tokens of each request's pages (a pool of just the pages that are written to)
        tail = [(q, q + (n - q) % page) for q, n in lengths]
        table, _, blocks = _pages(case, tail, gen, device, spare=16)
        starts = torch.tensor([0] + q_lens, device=device).cumsum(0)
        req = torch.arange(R, device=device).repeat_interleave(torch.tensor(q_lens, device=device))
        at = torch.arange(T, device=device) - starts[req] + torch.tensor([n - q for q, n in tail], device=device)[req]
        slots = table[req, at // page].long() * page + at % page
        slots = torch.cat([slots, slots.new_full((case["pad"],), -1)])   # padding tokens
        k_cache, v_cache = _caches(case, blocks, gen, device)
        kv = torch.randn((2, T + case["pad"], Hkv, D), generator=gen, device=device).to(_DTYPES[case["src"]])
        return dict(op="write", key=kv[0], value=kv[1], k_cache=k_cache, v_cache=v_cache, slots=slots)

    table, _, blocks = _pages(case, lengths, gen, device, spare=1)
    k_cache, v_cache = _caches(case, blocks, gen, device)
    q = torch.randn((T, Hq, D), generator=gen, device=device).to(_DTYPES[case["dtype"]])
    state = dict(op=case["op"], q=q, k_cache=k_cache, v_cache=v_cache, block_table=table, seq_lens=_int32(kv_lens, device),
                 scale=D ** -0.5, window=case["window"], longest=max(kv_lens), out=torch.zeros_like(q),
                 lse=torch.zeros((T, Hq), dtype=torch.float32, device=device),
                 workspace=torch.zeros(_WORKSPACE, dtype=torch.uint8, device=device))
    if case["op"] == "cross":
        state |= dict(query_start_loc=torch.tensor([0] + q_lens, device=device).cumsum(0).to(torch.int32), longest_q=max(q_lens))
    return state


def run(state):
    return _RUN[state["op"]](state)


def _run_tables(s):
    names = ("block_table", "seq_lens", "query_start_loc", "slot_mapping", "positions", "pages_taken")
    if own:
        from pth_flash_attn_b200 import ops
        ops.page_tables(s["context_lens"], s["query_lens"], s["free_blocks"], *(s[n] for n in names), s["page"])
        return {n: s[n] for n in names}
    page, free, table = s["page"], s["free_blocks"], s["block_table"]
    context, new_tokens = s["context_lens"].long(), s["query_lens"].long()
    seq_lens = context + new_tokens
    starts = torch.cat([new_tokens.new_zeros(1), new_tokens.cumsum(0)])
    old = (context + page - 1) // page
    new = (seq_lens + page - 1) // page - old
    first = new.cumsum(0) - new
    j = torch.arange(table.shape[1], device=table.device) - old[:, None]
    from_list = first[:, None] + j
    given = torch.where(from_list < len(free), free[from_list.clamp(0, len(free) - 1)], -1)
    table = torch.where((j >= 0) & (j < new[:, None]), given, table)
    t = torch.arange(len(s["slot_mapping"]), device=table.device)
    marks = torch.zeros(len(t) + 1, dtype=torch.int64, device=table.device)
    req = marks.index_add(0, starts[1:-1].clamp(max=len(t)), torch.ones_like(starts[1:-1])).cumsum(0)[:len(t)]
    live = t < starts[-1]
    at = torch.where(live, context[req] + t - starts[req], 0)
    block = table[req, (at // page).clamp(max=table.shape[1] - 1)].long()
    slots = torch.where(live & (block >= 0), block * page + at % page, -1)
    return dict(zip(names, (table, seq_lens.int(), starts.int(), slots, at, new.sum().int().reshape(1))))


def _run_write(s):
    if own:
        from pth_flash_attn_b200 import ops
        ops.kv16_write(s["key"], s["value"], s["k_cache"], s["v_cache"], s["slots"])
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    live = s["slots"] >= 0
    slots, page = s["slots"][live], s["k_cache"].shape[1]
    for name, rows in (("k_cache", s["key"]), ("v_cache", s["value"])):
        s[name][slots // page, slots % page] = rows[live].float().to(s[name].dtype)
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _run_decode(s):
    if own:
        from pth_flash_attn_b200 import ops
        ops.kv16_decode_attention(s["out"], s["lse"], s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["seq_lens"],
                                  s["scale"], s["workspace"], s["window"])
        return {"out": s["out"], "lse": s["lse"]}
    q, (R, Hq, D) = s["q"], s["q"].shape
    keys, values, seen = _gather(s)
    if s["window"]:
        seen &= torch.arange(seen.shape[1], device=q.device) >= (s["seq_lens"] - s["window"])[:, None]
    out, lse = _attend(q.float().view(R, -1, Hq // keys.shape[1], D), keys, values, seen, s["scale"])
    return {"out": out.reshape(R, Hq, D).to(q.dtype), "lse": lse.reshape(R, Hq)}


def _run_cross(s):
    if own:
        from pth_flash_attn_b200 import ops
        ops.kv16_cross_attention(s["out"], s["lse"], s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["seq_lens"],
                                 s["query_start_loc"], s["longest_q"], s["scale"], s["workspace"])
        return {"out": s["out"], "lse": s["lse"]}
    q, (T, Hq, D) = s["q"], s["q"].shape
    keys, values, seen = _gather(s)
    R, Hkv = keys.shape[:2]
    starts, G, n = s["query_start_loc"].long(), Hq // keys.shape[1], s["longest_q"]
    i = torch.arange(n, device=q.device)
    token, live = starts[:-1, None] + i, i < (starts[1:] - starts[:-1])[:, None]
    rows = q[token.clamp(max=T - 1)].float().view(R, n, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(R, Hkv, G * n, D)
    out, lse = _attend(rows, keys, values, seen, s["scale"])
    out = out.view(R, Hkv, G, n, D).permute(0, 3, 1, 2, 4).reshape(R, n, Hq, D)
    lse = lse.view(R, Hkv, G, n).permute(0, 3, 1, 2).reshape(R, n, Hq)
    return {"out": out[live].to(q.dtype), "lse": lse[live]}


def _gather(s):
    """Keys and values [R, Hkv, keys, D] of every request up to the longest, and which of them are its own."""
    page, table = s["k_cache"].shape[1], s["block_table"]
    at = torch.arange(s["longest"], device=table.device)
    block, slot = table[:, at // page].long(), at % page
    return (s["k_cache"][block, slot].float().transpose(1, 2), s["v_cache"][block, slot].float().transpose(1, 2),
            at < s["seq_lens"][:, None])


def _attend(rows, keys, values, seen, scale):
    """rows [R, Hkv, rows, D] over keys: the output and the log-sum-exp; a row that sees no key is 0 and -inf."""
    scores = (rows @ keys.transpose(2, 3)).mul_(scale).masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p @ values) / total.clamp(min=torch.finfo(torch.float32).tiny)
    return out, torch.where(total > 0, top + total.log(), -math.inf)[..., 0]


_RUN = {"tables": _run_tables, "write": _run_write, "decode": _run_decode, "cross": _run_cross}


def exact(case, seed):
    """The attention outputs and the written caches in 64 bits, request by request."""
    if case["op"] == "tables":
        return None   # whole numbers: there is nothing to round
    s = prepare(case, seed)
    page = s["k_cache"].shape[1]
    if case["op"] == "write":
        result = {}
        for name, rows in (("k_cache", s["key"]), ("v_cache", s["value"])):
            flat = s[name].double().reshape(-1, case["Hkv"], case["D"])
            kept = s["slots"] >= 0
            flat[s["slots"][kept]] = rows[kept].double()
            result[name] = flat.view(s[name].shape)
        return result
    G, D = case["Hq"] // case["Hkv"], case["D"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    first = 0
    for r, (q_len, n) in enumerate(_lengths(case)):
        tokens = slice(first, first + q_len)
        first += q_len
        low = max(0, n - case["window"]) if case["window"] else 0
        if n == 0 or q_len == 0:
            continue
        at = torch.arange(low, n, device="cuda")
        where = s["block_table"][r].long()[at // page], at % page
        for h in range(case["Hkv"]):
            heads = slice(h * G, (h + 1) * G)
            k, v = s["k_cache"][:, :, h][where].double(), s["v_cache"][:, :, h][where].double()
            scores = torch.einsum("thd,jd->thj", s["q"][tokens, heads].double(), k) / math.sqrt(D)
            lse[tokens, heads] = torch.logsumexp(scores, -1)
            out[tokens, heads] = torch.einsum("thj,jd->thd", torch.softmax(scores, -1), v)
    return {"out": out, "lse": lse}
